// The paged 4-bit key / value cache: rows in (spx_kv4_append), values out (spx_kv4_read) and
// attention over it (spx_kv4_attention). include/spx.h states the format and the pool's layout.
//
// The layout is the matrix cores': a tile of 16 tokens of one head is one contiguous run of
// 18 * head_dim bytes, in which each lane of a wave finds the codes that it feeds to the matrix
// instructions in one load. Scales have 8 significant bits, so integer * scale (at most 3 + 8
// bits, or 8 times the scale) is exact in f16 and the matrix cores read the values themselves.
#include <type_traits>

#include "batch.h"
#include "dev.h"

namespace spx {

typedef _Float16 h2v __attribute__((ext_vector_type(2)));
typedef _Float16 h8v __attribute__((ext_vector_type(8)));
typedef uint32_t u4v __attribute__((ext_vector_type(4)));

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

// A thread's piece of a row: eight channels of the key (kv = 0) or the value (1) of one head.
template <int HD>
struct Piece {
  int row, head, kv, c8;  // c8: channels 8 c8 ..
};
// Rows run fastest above the pieces of a row, so that a wave fills whole cache lines of a tile.
template <int HD>
__device__ __forceinline__ bool piece_of(const Kv4Rows &a, int64_t i, Piece<HD> &p) {
  constexpr int PC = HD / 8;
  p.c8 = (int)(i % PC);
  i /= PC;
  p.row = (int)(i % a.rows);
  i /= a.rows;
  p.kv = (int)(i & 1);
  p.head = (int)(i >> 1);
  return p.head < a.n_kv;
}

// ------------------------------------------------------------------ append
// The integer nearest to x / d, half to even, exactly: the quotient's estimate is off by at most
// one, and x - c d is exact (c d has at most 12 bits and is within a factor of two of x, or zero).
__device__ __forceinline__ int kv4_code(float x, float d, float inv) {
  float c = rintf(x * inv);
  c = fminf(fmaxf(c, -9.0f), 9.0f);
  const float e = fmaf(-c, d, x) * (d < 0.0f ? -1.0f : 1.0f), h = 0.5f * fabsf(d);  // e: the rest, in d's direction
  const bool odd = ((int)c & 1) != 0;
  if (e > h || (e == h && odd)) c += 1.0f;
  else if (e < -h || (e == -h && odd)) c -= 1.0f;
  return (int)fminf(fmaxf(c, -8.0f), 7.0f);
}

// A thread quantizes eight channels; the four threads of a quad share a group's scale.
// Bound by bytes: each value is read once (4 or 2 bytes) and 4.5 bits are written.
template <int HD, class R>
__global__ __launch_bounds__(256) void k_kv4_append(const Kv4Rows a) {
  typedef typename R::E E;
  Piece<HD> p;
  if (!piece_of<HD>(a, (int64_t)blockIdx.x * 256 + threadIdx.x, p)) return;
  int pg, t;
  if (!slot_of(a.slots[p.row], a.page, a.n_pages, pg, t)) return;  // (a quad has one row)
  const E *src = (p.kv ? (const E *)a.v + (int64_t)p.row * a.ld_v : (const E *)a.k + (int64_t)p.row * a.ld_k) + p.head * HD + p.c8 * 8;
  float x[8];
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < 8; j++) {
    x[j] = row_get(R{}, src[j]);
    m = max(m, __float_as_uint(x[j]) & 0x7fffffffu);  // magnitudes order as integers, NaN above all
  }
  m = max(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0xB1, 0xF, 0xF, true));
  m = max(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0x4E, 0xF, 0xF, true));
  // the first value of that magnitude gives the sign: place << 1 | negative, the smallest of all
  uint32_t key = ~0u;
#pragma unroll
  for (int j = 7; j >= 0; j--)
    if ((__float_as_uint(x[j]) & 0x7fffffffu) == m) key = (uint32_t)(((p.c8 & 3) * 8 + j) << 1) | (__float_as_uint(x[j]) >> 31);
  key = min(key, (uint32_t)__builtin_amdgcn_mov_dpp((int)key, 0xB1, 0xF, 0xF, true));
  key = min(key, (uint32_t)__builtin_amdgcn_mov_dpp((int)key, 0x4E, 0xF, 0xF, true));
  const bool bad = m >= 0x7f800000u;
  const float most = __uint_as_float(m | (key << 31));
  float d = row_get(RowBF16{}, bf16_rne(most * -0.125f));
  d = (float)(_Float16)fminf(fmaxf(d, -KV4_DMAX), KV4_DMAX) + 0.0f;  // (a scale of zero is +0)
  const float inv = d == 0.0f ? 0.0f : 1.0f / d;
  int c[8];
#pragma unroll
  for (int j = 0; j < 8; j++) c[j] = bad || d == 0.0f ? 8 : kv4_code(x[j], d, inv) + 8;
  const _Float16 dh = bad ? (_Float16)__builtin_nanf("") : (_Float16)d;
  constexpr int G = HD / 32;
  uint8_t *tile = a.pool + tile_at<HD>(pg, a.n_kv, p.head, a.page, t);
  const int ti = t & 15, g = p.c8 >> 2, h = p.c8 & 3;
  if (!p.kv) {
    uint32_t w = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) w |= (uint32_t)c[j] << (4 * ((j >> 1) + 4 * (j & 1)));
    *(uint32_t *)(tile + ((h * 16 + ti) * G + g) * 4) = w;
    if (h == 0) *(_Float16 *)(tile + 16 * HD + (ti * G + g) * 2) = dh;
  } else {
    uint32_t w = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) w |= (uint32_t)c[j] << (4 * j);
    uint8_t *vc = tile + 8 * HD + (ti >> 2) * 64 * G + (ti & 3) * G;
    if (HD == 128) {
      *(uint32_t *)(vc + p.c8 * 16) = w;
    } else {  // a lane of the attention kernels has four channels: two lanes' halves
      *(uint16_t *)(vc + (2 * p.c8) * 8) = (uint16_t)w;
      *(uint16_t *)(vc + (2 * p.c8 + 1) * 8) = (uint16_t)(w >> 16);
    }
    if (h == 0) *(_Float16 *)(tile + 17 * HD + (g * 16 + ti) * 2) = dh;
  }
}

// ------------------------------------------------------------------ read
template <int HD, class R>
__global__ __launch_bounds__(256) void k_kv4_read(const Kv4Rows a) {
  typedef typename R::E E;
  Piece<HD> p;
  if (!piece_of<HD>(a, (int64_t)blockIdx.x * 256 + threadIdx.x, p)) return;
  int pg, t;
  const bool in = slot_of(a.slots[p.row], a.page, a.n_pages, pg, t);
  E *dst = (p.kv ? (E *)a.v + (int64_t)p.row * a.ld_v : (E *)a.k + (int64_t)p.row * a.ld_k) + p.head * HD + p.c8 * 8;
  float x[8] = {};
  if (in) {
    constexpr int G = HD / 32;
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
#pragma unroll
  for (int j = 0; j < 8; j++) dst[j] = row_put(R{}, x[j]);
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

hipError_t launch_kv4_append(const Kv4Rows &a, int hd, int type, hipStream_t s) {
  const int64_t n = (int64_t)a.rows * a.n_kv * 2 * (hd / 8);
#define CALL(H, R) hipLaunchKernelGGL((k_kv4_append<H, R>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, a)
  KV4_BY_TYPE(hd, type, CALL)
#undef CALL
  return hipGetLastError();
}

hipError_t launch_kv4_read(const Kv4Rows &a, int hd, int type, hipStream_t s) {
  const int64_t n = (int64_t)a.rows * a.n_kv * 2 * (hd / 8);
#define CALL(H, R) hipLaunchKernelGGL((k_kv4_read<H, R>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, a)
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
// afterwards, with one multiply-add a token, row and group. Values become integer * scale in f16
// (exact): their scale belongs to the token, which the sum runs over.
//
// A query row is scaled by a power of two to fill f16's range; in two parts (SPX_F32) it has 22 bits.
// Probabilities are held relative to a running maximum, times 2^10, so that small ones keep their
// bits in f16; a maximum that grows by less than 2^5 leaves the reference as it is. In two parts
// (SPX_F32, SPX_F16) they have 22 bits too: one part's rounding (2^-11) would add to the output's own
// in SPX_F16; in SPX_BF16 it is an eighth of it.
constexpr float P_LIFT = 10.0f, P_SLACK = 5.0f;

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
// Eight codes of a key word as eight f16 values, channels in order: subnormals code * 2^-24 in
// elements 0, 1, 4, 5, code * 2^-20 in the others.
__device__ __forceinline__ h8v key_codes(uint32_t w, const Const4 &k) {
  const uint32_t w8 = w >> 8;
  const uint32_t x[4] = {w & k.lo, w & k.hi, w8 & k.lo, w8 & k.hi};
  return __builtin_bit_cast(h8v, x);
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

// The largest power of two that leaves |amax| at most 2^14 (1 for zero or what is not finite).
__device__ __forceinline__ float lift_of(float amax) {
  if (!(amax > 0.0f) || !(amax < __builtin_inff())) return 1.0f;
  int e;
  (void)frexpf(amax, &e);
  return ldexpf(1.0f, min(max(14 - e, -100), 100));
}

// Long sequences are shared by workgroups: chunk blockIdx.z of `chunk` tokens (and every
// gridDim.z-th after it). A workgroup leaves its rows' (maximum, sum, output) for k_kv4_join where
// there is more than one chunk to them.
template <int HD, class R, int QP, int PP>
__global__ __launch_bounds__(256) void k_kv4_attn(const Kv4Attn a) {
  typedef typename R::E E;
  constexpr int G = HD / 32, NC = HD / 16, NW = 4;
  __shared__ float so[NW][16][HD + 4], sm[NW][16], sl[NW][16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l = lane & 15, h = lane >> 4, head = blockIdx.y;
  Job4 j;
  if (!job_of<16>(a, blockIdx.x, j)) return;
  const int rows = j.nq * a.group, r = j.r0 + l, tok = min(r, rows - 1) / a.group, g0 = min(r, rows - 1) % a.group;
  // the row's query, its scale and what it sees
  const E *qp = (const E *)a.q + (int64_t)(j.q0 + tok) * a.ld_q + (head * a.group + g0) * HD + 8 * h;
  float qv[G][8], amax = 0.0f;
#pragma unroll
  for (int g = 0; g < G; g++)
#pragma unroll
    for (int i = 0; i < 8; i++) {
      qv[g][i] = row_get(R{}, qp[32 * g + i]);
      amax = fmaxf(amax, fabsf(qv[g][i]));
    }
  amax = max32(max16(amax));
  const float lift = lift_of(amax), unlift = a.scale / lift * 16777216.0f;
  h8v qh[G], ql[G];
  f4v zero[G];  // where a group's sum starts
#pragma unroll
  for (int g = 0; g < G; g++) {
    float all = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const float x = qv[g][i] * lift, down = i & 2 ? 0.0625f : 1.0f;
      const _Float16 top = (_Float16)x;
      const _Float16 low = (_Float16)(QP == 2 ? x - (float)top : 0.0f);
      all += (float)top + (float)low;
      qh[g][i] = (_Float16)((float)top * down);
      ql[g][i] = (_Float16)((float)low * down);
    }
    all = add32(add16(all)) * (-8.0f / 16777216.0f);
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
  float m = -__builtin_inff(), sum = 0.0f;
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
        const h8v kf = key_codes(x[u].k[g], kc);
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
    mt = max32(max16(mt)) * unlift;  // (unlift is positive)
    if (__builtin_amdgcn_ballot_w64(mt > m + P_SLACK)) {
      const float mn = fmaxf(m, mt), f = m == mn ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
      m = mn;
      sum *= f;
#pragma unroll
      for (int c = 0; c < NC; c++) o[c] *= f;
    }
    const float ref = m == -__builtin_inff() ? 0.0f : P_LIFT - m;
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
  if (h == 0) { sm[wave][l] = m; sl[wave][l] = sum; }
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
    for (int c = 0; c < NC; c++) dst[c] = row_put(R{}, v[c] * inv);
    return;
  }
  const int64_t at = (((int64_t)blockIdx.x * a.n_kv + head) * gridDim.z + blockIdx.z) * 16 + row;
  float *dst = a.part + at * HD + part * NC;
#pragma unroll
  for (int c = 0; c < NC; c += 4) *(float4 *)(dst + c) = make_float4(v[c], v[c + 1], v[c + 2], v[c + 3]);
  if (part == 0) ((float2 *)(a.part + (int64_t)gridDim.x * a.n_kv * gridDim.z * 16 * HD))[at] = make_float2(mm, total);
}

// The chunks of a job's rows together: a wave has four rows, 16 lanes each.
template <int HD, class R>
__global__ __launch_bounds__(64) void k_kv4_join(const Kv4Attn a, int splits) {
  typedef typename R::E E;
  constexpr int NC = HD / 16, U = 4;
  Job4 j;
  if (!job_of<16>(a, blockIdx.x, j)) return;
  const int rows = j.nq * a.group, head = blockIdx.y, row = blockIdx.z * 4 + (threadIdx.x >> 4), part = threadIdx.x & 15, rr = j.r0 + row;
  const int last = min(j.r0 + 15, rows - 1) / a.group, first = j.r0 / a.group;
  const int all_hi = min(j.n - j.nq + last + 1, j.n), from = (a.window > 0 ? max(j.n - j.nq + first + 1 - a.window, 0) : 0) & ~31;
  const int n = min(all_hi > from ? (all_hi - from + a.chunk - 1) / a.chunk : 1, splits);
  if (n == 1 || rr >= rows) return;
  const int64_t at = ((int64_t)blockIdx.x * a.n_kv + head) * splits * 16 + row;
  const float2 *ms = (const float2 *)(a.part + (int64_t)gridDim.x * a.n_kv * splits * 16 * HD) + at;
  const float *src = a.part + at * HD + part * NC;
  float m = -__builtin_inff();
  for (int c = part; c < n; c += 16) m = fmaxf(m, ms[c * 16].x);
  m = fmaxf(m, SPX_DPPF(m, 0xB1));
  m = fmaxf(m, SPX_DPPF(m, 0x4E));
  m = fmaxf(m, SPX_DPPF(m, 0x141));
  m = fmaxf(m, SPX_DPPF(m, 0x140));
  float total = 0.0f, v[NC] = {};
  for (int c0 = 0; c0 < n; c0 += U) {  // U chunks' loads at a time
    float2 x[U];
    float4 y[U][NC / 4];
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int c = min(c0 + u, n - 1);
      x[u] = ms[c * 16];
#pragma unroll
      for (int i = 0; i < NC / 4; i++) y[u][i] = *(const float4 *)(src + (int64_t)c * 16 * HD + 4 * i);
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
      const float f = x[u].x == m ? 1.0f : __builtin_amdgcn_exp2f(x[u].x - m);
      if (c0 + u >= n) continue;  // (0 times a NaN is one)
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
  const float inv = total == 0.0f ? 0.0f : 1.0f / total;
  E *dst = (E *)a.out + (int64_t)(j.q0 + rr / a.group) * a.ld_out + (head * a.group + rr % a.group) * HD + part * NC;
#pragma unroll
  for (int i = 0; i < NC; i++) dst[i] = row_put(R{}, v[i] * inv);
}

// How the work is split: jobs, chunks of a sequence (at most) and tokens a chunk. Chunks are as long
// as leaves about KV4_WGS workgroups, 128 tokens (a tile a wave) at least.
constexpr int KV4_WGS = 2048;
struct Split4 { int64_t jobs; int splits, chunk; };
static Split4 split_of(int group, int n_kv, int rows, int n_seq, int max_kv) {
  Split4 r;
  r.jobs = (int64_t)rows * group / 16 + n_seq;
  const int64_t busy = (((int64_t)rows * group + n_seq - 1) / n_seq + 15) / 16 * n_seq * n_kv;  // jobs with rows, all key heads
  const int64_t want = (KV4_WGS + busy - 1) / busy;
  int64_t chunk = ((max_kv + want - 1) / want + 127) / 128 * 128;
  if (chunk < 128) chunk = 128;
  if (chunk > 1 << 20) chunk = 1 << 20;
  r.chunk = (int)chunk;
  r.splits = (int)((max_kv + chunk - 1) / chunk);
  if (r.splits < 1) r.splits = 1;
  return r;
}
int64_t kv4_attention_ws(int hd, int group, int n_kv, int rows, int n_seq, int max_kv) {
  const Split4 d = split_of(group, n_kv, rows, n_seq, max_kv);
  return d.splits > 1 ? (d.jobs | 1) * n_kv * d.splits * 16 * (hd + 2) * 4 : 0;
}

hipError_t launch_kv4_attention(Kv4Attn a, int hd, int type, int max_kv, hipStream_t s) {
  const Split4 d = split_of(a.group, a.n_kv, a.rows, a.n_seq, max_kv);
  a.chunk = d.chunk;
  // an odd count, so that neighbouring key heads and chunks of a sequence go to other XCDs (workgroups go
  // around the eight of them in order)
  const dim3 grid((unsigned)d.jobs | 1, (unsigned)a.n_kv, (unsigned)d.splits);
#define CALL(H, R)                                                                                                              \
  hipLaunchKernelGGL((k_kv4_attn<H, R, sizeof(R::E) == 4 ? 2 : 1, std::is_same<R, RowBF16>::value ? 1 : 2>), grid, dim3(256), 0, \
                     s, a);                                                                                                     \
  if (d.splits > 1) hipLaunchKernelGGL((k_kv4_join<H, R>), dim3(grid.x, grid.y, 4), dim3(64), 0, s, a, d.splits)
  KV4_BY_TYPE(hd, type, CALL)
#undef CALL
  return hipGetLastError();
}

}  // namespace spx
