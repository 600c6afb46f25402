// A mixture of experts over a batch: the router's choice and its gradient, rows sorted by expert, gathered,
// joined again and that gradient (spx_moe_route .. spx_moe_combine_grad).
#include <algorithm>
#include <type_traits>

#include "dev.h"
#include "experts.h"
#include "rows.h"

namespace spx {

// ------------------------------------------------------------------ the router
// A wave has a row, its lane l the logits l, l + 64, ...; NV of them. 8191 rows of 128 logits take 6.2 us, eight rounds of
// a maximum across the wave (ten instructions that wait for each other) being most of it, the gradient 6.1; their bytes 1 and
// 2 us. 24 rows take 3.5 us, little more than a launch.

// Logits' order as numbers: larger logit, larger number; -0 as 0; NaN above all. 0: none.
__device__ __forceinline__ uint32_t logit_key(float v) {
  const uint32_t u = __float_as_uint(v + 0.0f);
  if ((u & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

template <class R, int NV>
__device__ __forceinline__ void route_logits(const RouteArgs &a, int row, float (&x)[NV]) {
  const int lane = threadIdx.x & 63;
  const typename R::E *src = (const typename R::E *)a.logits + (int64_t)row * a.ld;
#pragma unroll
  for (int v = 0; v < NV; v++) {
    const int e = lane + 64 * v;
    x[v] = e < a.n_expert ? row_get(R{}, src[e]) : -INFINITY;
  }
}

// k rounds of: the wave's largest key, the lowest id that holds it. Lane i keeps the i-th.
template <class R, int NV>
__global__ __launch_bounds__(256) void k_moe_route(const RouteArgs a) {
  const int row = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (row >= a.rows) return;
  float x[NV];
  route_logits<R, NV>(a, row, x);
  uint32_t key[NV];
#pragma unroll
  for (int v = 0; v < NV; v++) key[v] = lane + 64 * v < a.n_expert ? logit_key(x[v]) : 0u;
  int my_e = 0;
  float my_x = 0.0f, m = 0.0f;
  for (int i = 0; i < a.k; i++) {
    uint32_t best = key[0];
#pragma unroll
    for (int v = 1; v < NV; v++) best = max(best, key[v]);
    best = wave_max_u32(best);
    int e = 0;
    float at = 0.0f;
#pragma unroll
    for (int v = NV - 1; v >= 0; v--) {
      const unsigned long long holds = __builtin_amdgcn_ballot_w64(key[v] == best);
      if (holds) {
        const int l = (int)__builtin_ctzll(holds);
        e = 64 * v + l;
        at = lane_f(x[v], l);
      }
    }
    if (i == 0) m = at;
    if (lane == i) { my_e = e; my_x = at; }
#pragma unroll
    for (int v = 0; v < NV; v++)
      if (lane + 64 * v == e) key[v] = 0u;
  }
  // m is the row's maximum, or a NaN if it holds one. -inf: nothing is likely, weights are 0.
  const float p = lane < a.k && m != -INFINITY ? expf(my_x - m) : 0.0f;
  float total = 0.0f;
  if (a.norm) total = p;
  else
#pragma unroll
    for (int v = 0; v < NV; v++) total += expf(x[v] - m);
  total = wave_sum(total);
  if (lane < a.k) {
    a.chosen[(int64_t)row * a.k + lane] = my_e;
    a.weights[(int64_t)row * a.k + lane] = m == -INFINITY ? 0.0f : p / total;
  }
}

// With w the weights and g their gradient, s = sum w g: d x_c = w_c (g_c - s), where the weights are over all
// experts also d x_e = -p_e s of the others. Lane i holds the i-th chosen id, its weight and gradient.
template <class R, int NV>
__global__ __launch_bounds__(256) void k_moe_route_grad(const RouteArgs a) {
  const int row = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (row >= a.rows) return;
  typedef typename R::E E;
  float x[NV];
  route_logits<R, NV>(a, row, x);
  bool bad = false;
  float m = -INFINITY;
#pragma unroll
  for (int v = 0; v < NV; v++) {
    bad |= isnan(x[v]) || x[v] == INFINITY;
    m = fmaxf(m, x[v]);
  }
  m = wave_max(m);
  int id = -1;
  float g = 0.0f, xc = -INFINITY;
  if (lane < a.k) {
    id = a.chosen[(int64_t)row * a.k + lane];
    g = a.d_weights[(int64_t)row * a.k + lane];
    bad |= id < 0 || id >= a.n_expert;
    if (id >= 0 && id < a.n_expert) xc = row_get(R{}, ((const E *)a.logits)[(int64_t)row * a.ld + id]);
  }
  bad = __builtin_amdgcn_ballot_w64(bad) != 0;
  const float mc = a.norm ? wave_max(xc) : m;  // (the weights' own maximum, whatever ids are given)
  const float pc = xc == -INFINITY ? 0.0f : expf(xc - mc);
  float p[NV], total = pc;
  if (!a.norm) {
    total = 0.0f;
#pragma unroll
    for (int v = 0; v < NV; v++) { p[v] = x[v] == -INFINITY ? 0.0f : expf(x[v] - m); total += p[v]; }
  }
  total = wave_sum(total);
  const float inv = total > 0.0f ? 1.0f / total : 0.0f, w = pc * inv, s = wave_sum(lane < a.k ? w * g : 0.0f);
  const float mine = a.norm ? w * (g - s) : w * g;
  E *out = (E *)a.d_logits + (int64_t)row * a.ld_d;
  float d[NV];
#pragma unroll
  for (int v = 0; v < NV; v++) d[v] = a.norm ? 0.0f : -(p[v] * inv) * s;
  for (int j = 0; j < a.k; j++) {
    const int e = lane_i(id, j);
    const float add = lane_f(mine, j);
#pragma unroll
    for (int v = 0; v < NV; v++)
      if (lane + 64 * v == e) d[v] += add;
  }
#pragma unroll
  for (int v = 0; v < NV; v++)
    if (lane + 64 * v < a.n_expert) out[lane + 64 * v] = row_put(R{}, bad ? __builtin_nanf("") : m == -INFINITY ? 0.0f : d[v]);  // (-inf: whatever g is)
}

#define MOE_BY_TYPE(type, CALL)               \
  switch (type) {                             \
  case T_F32: { CALL(RowF32); break; }        \
  case T_F16: { CALL(RowF16); break; }        \
  case T_BF16: { CALL(RowBF16); break; }      \
  default: return hipErrorInvalidValue;       \
  }

template <class R>
static void route(const RouteArgs &a, bool grad, hipStream_t s) {
  const dim3 grid((unsigned)(a.rows + 3) / 4), block(256);
#define ROUTE(NV)                                                                              \
  if (grad) hipLaunchKernelGGL((k_moe_route_grad<R, NV>), grid, block, 0, s, a);               \
  else hipLaunchKernelGGL((k_moe_route<R, NV>), grid, block, 0, s, a)
  if (a.n_expert <= 64) { ROUTE(1); }
  else if (a.n_expert <= 128) { ROUTE(2); }
  else if (a.n_expert <= 256) { ROUTE(4); }
  else if (a.n_expert <= 512) { ROUTE(8); }
  else { ROUTE(16); }
#undef ROUTE
}
hipError_t launch_moe_route(const RouteArgs &a, int type, hipStream_t s) {
#define CALL(R) route<R>(a, false, s)
  MOE_BY_TYPE(type, CALL)
#undef CALL
  return hipGetLastError();
}
hipError_t launch_moe_route_grad(const RouteArgs &a, int type, hipStream_t s) {
#define CALL(R) route<R>(a, true, s)
  MOE_BY_TYPE(type, CALL)
#undef CALL
  return hipGetLastError();
}

// ------------------------------------------------------------------ sorting by expert
// A counting sort that keeps the order of equal ones. A workgroup has a run of entries, each of its waves
// a run of those; entries of no expert are those of a last, (n_expert + 1)-th bucket. An entry's place is its
// bucket's start, plus the bucket's entries in earlier workgroups, in the workgroup's earlier waves, earlier in the
// wave's run and at lower lanes. Counts are sums of integers: no order of additions changes them. Up to 4096 entries are one
// workgroup's (192 entries 3.9 us), more have a launch that counts before (65528 entries 4.8 + 5.7 us): both bound by launches and
// dependent steps, not by their 0.8 MB.
constexpr int SORT_T = 512, SORT_W = SORT_T / 64;
constexpr int SORT_ALONE = 4096;  // so many entries are one workgroup's

static int sort_run(int64_t n) {  // a workgroup's entries
  if (n <= SORT_ALONE) return SORT_ALONE;
  const int64_t per = ((n + 255) / 256 + SORT_T - 1) / SORT_T * SORT_T;
  return (int)(per < 2 * SORT_T ? 2 * SORT_T : per);
}
int moe_sort_blocks(int64_t n) { return (int)((n + sort_run(n) - 1) / sort_run(n)); }

__device__ __forceinline__ int bucket_of(const SortArgs &a, int i) {
  const int e = a.chosen[i];
  return e >= 0 && e < a.n_expert ? e : a.n_expert;
}

__global__ __launch_bounds__(SORT_T) void k_moe_count(const SortArgs a, int run) {
  __shared__ int count[MOE_MAX_E + 1];
  const int nb = a.n_expert + 1;
  for (int e = threadIdx.x; e < nb; e += SORT_T) count[e] = 0;
  __syncthreads();
  const int begin = blockIdx.x * run, end = min(begin + run, a.n);
  for (int i = begin + threadIdx.x; i < end; i += SORT_T) atomicAdd(&count[bucket_of(a, i)], 1);
  __syncthreads();
  for (int e = threadIdx.x; e < nb; e += SORT_T) a.counts[(int64_t)blockIdx.x * nb + e] = count[e];
}

__global__ __launch_bounds__(SORT_T) void k_moe_place(const SortArgs a, int run) {
  extern __shared__ int at[];  // [SORT_W][n_expert + 1]: counts, then the next place of each bucket
  __shared__ int up[SORT_W];
  const int t = threadIdx.x, wave = t >> 6, lane = t & 63, nb = a.n_expert + 1;
  for (int i = t; i < SORT_W * nb; i += SORT_T) at[i] = 0;
  __syncthreads();
  const int begin = blockIdx.x * run + wave * (run / SORT_W), end = min(begin + run / SORT_W, a.n);
  int *mine = at + wave * nb;
  for (int i = begin + lane; i < end; i += 64) atomicAdd(&mine[bucket_of(a, i)], 1);
  __syncthreads();
  int carry = 0;
  for (int b = 0; b < nb; b += SORT_T) {  // a thread a bucket
    const int e = b + t;
    int before = 0, all = 0;
    if (e < nb) {
      if (gridDim.x == 1) {
        for (int w = 0; w < SORT_W; w++) all += at[w * nb + e];
      } else {
#pragma unroll 16
        for (int g = 0; g < (int)gridDim.x; g++) {  // (sixteen loads under way: 64 workgroups 5.7 us, one by one 19)
          const int c = a.counts[(int64_t)g * nb + e];
          all += c;
          before += g < (int)blockIdx.x ? c : 0;
        }
      }
    }
    const int sum = wave_scan(all);
    if (lane == 63) up[wave] = sum;
    __syncthreads();
    int start = carry + sum - all;
    for (int w = 0; w < SORT_W; w++) {
      if (w < wave) start += up[w];
      carry += up[w];
    }
    if (e < nb) {
      if (blockIdx.x == 0) a.starts[e] = start;  // (the last bucket's: where the entries of experts end)
      int next = start + before;
      for (int w = 0; w < SORT_W; w++) {
        const int c = at[w * nb + e];
        at[w * nb + e] = next;
        next += c;
      }
    }
    __syncthreads();
  }
  const int bits = 32 - __builtin_clz(nb - 1);
  for (int i = begin + lane; i - lane < end; i += 64) {
    const bool in = i < end;
    const int e = in ? bucket_of(a, i) : 0;
    unsigned long long same = __builtin_amdgcn_ballot_w64(in);
    for (int b = 0; b < bits; b++) {
      const unsigned long long set = __builtin_amdgcn_ballot_w64((e >> b & 1) != 0);
      same &= e >> b & 1 ? set : ~set;
    }
    const unsigned long long lower = same & ((1ull << lane) - 1ull);
    const int p = in ? mine[e] + __builtin_popcountll(lower) : 0;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    if (in && (same >> lane) == 1ull) mine[e] = p + 1;  // the last of them
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    if (in) {
      const bool none = e == a.n_expert;
      a.order[p] = none ? -1 : i;
      a.place[i] = none ? -1 : p;
    }
  }
}

hipError_t launch_moe_sort(const SortArgs &a, hipStream_t s) {
  const int run = sort_run(a.n), blocks = a.n > 0 ? moe_sort_blocks(a.n) : 1;
  if (blocks > 1) hipLaunchKernelGGL(k_moe_count, dim3(blocks), dim3(SORT_T), 0, s, a, run);
  hipLaunchKernelGGL(k_moe_place, dim3(blocks), dim3(SORT_T), SORT_W * (a.n_expert + 1) * sizeof(int), s, a, run);
  return hipGetLastError();
}

// ------------------------------------------------------------------ rows there and back
// A power of two of threads has a row, each piece of it 16 bytes (VEC: all rows lie at multiples of 16 bytes
// and are as long) or one element.
template <class R, bool VEC>
struct RowPiece {
  typedef typename R::E E;
  static constexpr int N = VEC ? 16 / (int)sizeof(E) : 1;
  static __device__ __forceinline__ void get(const E *p, float (&x)[N]) {
    alignas(16) E e[N];
    if constexpr (VEC) *(uint4 *)e = *(const uint4 *)p;
    else e[0] = *p;
#pragma unroll
    for (int i = 0; i < N; i++) x[i] = row_get(R{}, e[i]);
  }
  static __device__ __forceinline__ void put(E *p, const float (&x)[N]) {
    alignas(16) E e[N];
#pragma unroll
    for (int i = 0; i < N; i++) e[i] = row_put(R{}, x[i]);
    if constexpr (VEC) *(uint4 *)p = *(const uint4 *)e;
    else *p = e[0];
  }
};

// Bound by its bytes, most of them out, which go past the caches and leave these to x (read k times); two rows a thread, so
// that their entries and then their pieces are under way together. Without weights a piece is copied as it is. 1024 rows of 2048
// in bf16, eight places each (38 MB): 6.9 us.
constexpr int GATHER_ROWS = 2;
// A piece of a row, times w where there are weights.
template <class R, bool WEIGHTED, int N, class Piece>
__device__ __forceinline__ Piece gathered(Piece v, float w) {
  if constexpr (WEIGHTED) {
    alignas(16) typename R::E e[N];
    *(Piece *)e = v;
#pragma unroll
    for (int j = 0; j < N; j++) e[j] = row_put(R{}, row_get(R{}, e[j]) * w);
    v = *(const Piece *)e;
  }
  return v;
}
template <class R, bool VEC, bool WEIGHTED>
__global__ __launch_bounds__(256) void k_moe_gather(const JoinArgs a, int log_t) {
  typedef RowPiece<R, VEC> P;
  typedef typename R::E E;
  typedef typename std::conditional<VEC, i4v, E>::type Piece;
  const int each = 256 >> log_t, i0 = blockIdx.x * (each * GATHER_ROWS) + (threadIdx.x >> log_t), t = threadIdx.x & ((1 << log_t) - 1);
  const int n = a.rows * a.k;
  const E *src[GATHER_ROWS];
  float w[GATHER_ROWS];
  bool is[GATHER_ROWS];
  int entry[GATHER_ROWS];
#pragma unroll
  for (int r = 0; r < GATHER_ROWS; r++) entry[r] = a.order[min(i0 + r * each, n - 1)];
#pragma unroll
  for (int r = 0; r < GATHER_ROWS; r++) {
    is[r] = entry[r] >= 0 && entry[r] < n;
    src[r] = (const E *)a.x + (int64_t)(is[r] ? entry[r] / a.k : 0) * a.ld_x;
    w[r] = WEIGHTED && is[r] ? a.weights[entry[r]] : 1.0f;
  }
  for (int c = t; c < a.width / P::N; c += 1 << log_t) {
    Piece v[GATHER_ROWS];
#pragma unroll
    for (int r = 0; r < GATHER_ROWS; r++) v[r] = *(const Piece *)(src[r] + c * P::N);
#pragma unroll
    for (int r = 0; r < GATHER_ROWS; r++) {
      const int i = i0 + r * each;
      if (i >= n) break;
      v[r] = is[r] ? gathered<R, WEIGHTED, P::N>(v[r], w[r]) : Piece{};
      Piece *const to = (Piece *)((E *)a.out + (int64_t)i * a.ld_out + c * P::N);
      if constexpr (VEC) __builtin_nontemporal_store(v[r], to);
      else *to = v[r];
    }
  }
}

// The same in an order that lets a row of x come once from memory and the other times from an L2: workgroups go to the XCDs in
// turn, and workgroup id has a slice of x's rows, about 2 MB, that is id % 8 of eight slices which are at work together. Of its
// part of the places it picks those that are the slice's (a place of no entry is any one slice's), and its waves have four of their
// rows each at a time. Its part is lines of 16 places from all over, the j-th turned by j times 0.618 of their number: places of
// one slice stand together in each expert's, and even strides would give some workgroups all of them.
// 8191 rows of 2048 in bf16, eight places each (302 MB): 57-59 us against 73 as above (four rows a thread there 75, eight 76, one 73);
// 32768 rows 204 us against 298, 4097 of 1024 in fp32 29 against 35, 16384 of 512 in bf16 26 against 35; 2048 rows of 2048 (8 MB of x) 18 against
// 17. Slices of 1 MB 59, of 4 MB 64; 16 places a workgroup on average 57, and 31 for the 4097 rows; a row a wave 62.
constexpr int NEAR_LINE = 16, NEAR_RUN = 2048, NEAR_AVERAGE = 12;  // (a run is NEAR_AVERAGE places for each slice: a multiple of NEAR_LINE)
constexpr int64_t NEAR_SLICE = 2200000;                            // bytes of x
// Its gain is what is not read again, k - 1 of k times x, which has to be worth its searches: in us, here / as above,
// rows of 2048 in bf16    3200: k 2 9.5 / 6.9, k 3 12.7 / 11.0;  8191: k 1 13.4 / 10.2, k 2 19.2 / 20.2, k 4 32 / 38;  16000: k 2 36.7 / 37.8, k 3 48 / 56
// rows of 1024 in fp32    4097: k 2 10.8 / 9.5, k 3 13.1 / 14.9, k 8 29 / 36
// rows of 512, 25 MB      k 2 12.6 / 15.2;  102 MB: k 1 34 / 31, k 2 50 / 59, k 8 161 / 228
// With weights the waves' four rows wait for a conversion between loads and stores, the longer the rows: 8191 rows of 4 KB k 2 25.9 / 20.5, k 4 42.5 / 37.9,
// k 6 54.9 / 55.6, k 8 69.8 / 73.5; 60000 rows of 1 KB k 2 33 / 36, k 4 51 / 71; 30000 rows of 2 KB k 2 41.7 / 37.0, k 3 51.4 / 53.0, k 8 97 / 136.
// (What the order holds is not known here: where seven of eight places have no entry, 30000 rows of 1024 in bf16 take 96 us with k = 8, 90 as above.)
static bool gather_near(int64_t rows, int k, int64_t row_bytes, bool weights) {
  return rows * row_bytes * (k - 1) > 11000000ll * k && (!weights || k >= (row_bytes > 2048 ? 6 : 3));
}
template <class R, bool WEIGHTED>
__global__ __launch_bounds__(256) void k_moe_gather_near(const JoinArgs a, int slices, int per, int run, int runs) {
  typedef typename R::E E;
  constexpr int N = 16 / (int)sizeof(E), U = 4;
  __shared__ int2 list[NEAR_RUN];  // places and their entries
  __shared__ int count;
  const int n = a.rows * a.k, t = threadIdx.x, wave = t >> 6, lane = t & 63, at = blockIdx.x >> 3, mine = at % runs;
  const int slice = at / runs * 8 + (blockIdx.x & 7), turn = (int)(0.618f * runs);
  if (t == 0) count = 0;
  __syncthreads();
  const int lo = (int)min((int64_t)slice * per, (int64_t)a.rows) * a.k, hi = (int)min((int64_t)(slice + 1) * per, (int64_t)a.rows) * a.k;
  for (int j = t; j < run; j += 256) {
    const int line = j / NEAR_LINE, i = (line * runs + (int)((uint32_t)(mine + line * turn) % (uint32_t)runs)) * NEAR_LINE + j % NEAR_LINE;
    if (i >= n) continue;
    const int entry = a.order[i];
    const bool is = entry >= 0 && entry < n;
    if (is ? entry >= lo && entry < hi : i / NEAR_LINE % slices == slice) list[atomicAdd(&count, 1)] = make_int2(i, is ? entry : -1);
  }
  __syncthreads();
  const int many = count, pieces = a.width / N;
  for (int q = wave * U; q < many; q += 4 * U) {
    const i4v *src[U];
    i4v *to[U];
    float w[U];
    bool is[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int at = min(q + u, many - 1), i = __builtin_amdgcn_readfirstlane(list[at].x), entry = __builtin_amdgcn_readfirstlane(list[at].y);
      is[u] = entry >= 0;
      src[u] = (const i4v *)((const E *)a.x + (int64_t)(max(entry, 0) / a.k) * a.ld_x);
      to[u] = (i4v *)((E *)a.out + (int64_t)i * a.ld_out);
      w[u] = WEIGHTED && is[u] ? a.weights[entry] : 1.0f;
    }
    for (int c = lane; c < pieces; c += 64) {
      i4v v[U];
#pragma unroll
      for (int u = 0; u < U; u++) v[u] = src[u][c];
#pragma unroll
      for (int u = 0; u < U; u++)
        if (q + u < many) __builtin_nontemporal_store(is[u] ? gathered<R, WEIGHTED, N>(v[u], w[u]) : i4v{}, to[u] + c);
    }
  }
}

// Bound by its bytes, most of them in; eight places at a time, so that their pieces are under way together. The same
// rows, 302 MB: 56 us (four at a time 81), 5.4 TB/s.
template <class R, bool VEC>
__global__ __launch_bounds__(256) void k_moe_combine(const JoinArgs a, int log_t) {
  typedef RowPiece<R, VEC> P;
  typedef typename R::E E;
  constexpr int J = 8;
  const int r = blockIdx.x * (256 >> log_t) + (threadIdx.x >> log_t), t = threadIdx.x & ((1 << log_t) - 1);
  if (r >= a.rows) return;
  const int n = a.rows * a.k;
  for (int c = t; c < a.width / P::N; c += 1 << log_t) {
    float sum[P::N] = {};
    for (int j0 = 0; j0 < a.k; j0 += J) {
      int p[J];
      float w[J], x[J][P::N];
#pragma unroll
      for (int j = 0; j < J; j++) {
        p[j] = j0 + j < a.k ? a.place[(int64_t)r * a.k + j0 + j] : -1;
        w[j] = a.weights && j0 + j < a.k ? a.weights[(int64_t)r * a.k + j0 + j] : 1.0f;
      }
#pragma unroll
      for (int j = 0; j < J; j++) P::get((const E *)a.x + (p[j] >= 0 && p[j] < n ? p[j] : 0) * a.ld_x + c * P::N, x[j]);
#pragma unroll
      for (int j = 0; j < J; j++) {
        const bool is = p[j] >= 0 && p[j] < n;
#pragma unroll
        for (int i = 0; i < P::N; i++) sum[i] = is ? fmaf(w[j], x[j][i], sum[i]) : sum[i];
      }
    }
    P::put((E *)a.out + (int64_t)r * a.ld_out + c * P::N, sum);
  }
}

// A wave has an entry: its row's d_out against its sorted row of y. (4097 rows of 1024 in fp32, eight places: 49 us, 285 MB, 5.8 TB/s;
// d_out is read eight times, seven of them from the caches.)
template <class R, bool VEC>
__global__ __launch_bounds__(256) void k_moe_combine_grad(const JoinArgs a) {
  typedef RowPiece<R, VEC> P;
  typedef typename R::E E;
  const int entry = blockIdx.x * 4 + (threadIdx.x >> 6), t = threadIdx.x & 63, n = a.rows * a.k;
  if (entry >= n) return;
  const int p = a.place[entry];
  const bool is = p >= 0 && p < n;
  float dot = 0.0f;
  if (is) {
    const float w = a.weights[entry];
    const E *d = (const E *)a.d + (int64_t)(entry / a.k) * a.ld_d, *y = (const E *)a.x + (int64_t)p * a.ld_x;
    E *out = (E *)a.out + (int64_t)p * a.ld_out;
    for (int c = t; c < a.width / P::N; c += 64) {
      float u[P::N], v[P::N];
      P::get(d + c * P::N, u);
      P::get(y + c * P::N, v);
#pragma unroll
      for (int i = 0; i < P::N; i++) {
        dot = fmaf(u[i], v[i], dot);
        u[i] *= w;
      }
      P::put(out + c * P::N, u);
    }
  }
  dot = wave_sum(dot);
  if (t == 0) a.d_weights[entry] = dot;
  const int none = a.order[entry];  // (as a place)
  if (none < 0 || none >= n) {
    E *out = (E *)a.out + (int64_t)entry * a.ld_out;
    const float zero[P::N] = {};
    for (int c = t; c < a.width / P::N; c += 64) P::put(out + c * P::N, zero);
  }
}

// Whether rows at p, ld apart, lie at multiples of 16 bytes.
static bool on16(const void *p, int64_t ld, int size) { return (uintptr_t)p % 16 == 0 && ld * size % 16 == 0; }

template <class R>
static void join(const JoinArgs &a, int what, hipStream_t s) {
  constexpr int size = sizeof(typename R::E);
  const bool vec = a.width * size % 16 == 0 && on16(a.x, a.ld_x, size) && on16(a.out, a.ld_out, size) && (what != 2 || on16(a.d, a.ld_d, size));
  const int pieces = vec ? a.width * size / 16 : a.width;
  int log_t = 0;
  while (log_t < 8 && (1 << log_t) < pieces) log_t++;
  const int rows = what == 0 ? a.rows * a.k : a.rows, each = (256 >> log_t) * (what == 0 ? GATHER_ROWS : 1);
  const dim3 grid((unsigned)((rows + each - 1) / each)), block(256);
  if (what == 0) {
    if (vec && pieces >= 64 && gather_near(a.rows, a.k, (int64_t)a.width * size, a.weights != nullptr)) {
      const int64_t bytes = (int64_t)a.rows * a.width * size;
      const int slices = 8 * (int)std::min<int64_t>((bytes + 8 * NEAR_SLICE - 1) / (8 * NEAR_SLICE), NEAR_RUN / (8 * NEAR_AVERAGE));
      const int run = NEAR_AVERAGE * slices, runs = (rows + run - 1) / run, per = (a.rows + slices - 1) / slices;
      const dim3 near((unsigned)(slices * runs));
      if (a.weights) hipLaunchKernelGGL((k_moe_gather_near<R, true>), near, block, 0, s, a, slices, per, run, runs);
      else hipLaunchKernelGGL((k_moe_gather_near<R, false>), near, block, 0, s, a, slices, per, run, runs);
    } else if (vec && a.weights) hipLaunchKernelGGL((k_moe_gather<R, true, true>), grid, block, 0, s, a, log_t);
    else if (vec) hipLaunchKernelGGL((k_moe_gather<R, true, false>), grid, block, 0, s, a, log_t);
    else if (a.weights) hipLaunchKernelGGL((k_moe_gather<R, false, true>), grid, block, 0, s, a, log_t);
    else hipLaunchKernelGGL((k_moe_gather<R, false, false>), grid, block, 0, s, a, log_t);
  } else if (what == 1) {
    if (vec) hipLaunchKernelGGL((k_moe_combine<R, true>), grid, block, 0, s, a, log_t);
    else hipLaunchKernelGGL((k_moe_combine<R, false>), grid, block, 0, s, a, log_t);
  } else {
    const dim3 waves((unsigned)((a.rows * a.k + 3) / 4));
    if (vec) hipLaunchKernelGGL((k_moe_combine_grad<R, true>), waves, block, 0, s, a);
    else hipLaunchKernelGGL((k_moe_combine_grad<R, false>), waves, block, 0, s, a);
  }
}
static hipError_t launch_join(const JoinArgs &a, int type, int what, hipStream_t s) {
#define CALL(R) join<R>(a, what, s)
  MOE_BY_TYPE(type, CALL)
#undef CALL
  return hipGetLastError();
}
hipError_t launch_moe_gather(const JoinArgs &a, int type, hipStream_t s) { return launch_join(a, type, 0, s); }
hipError_t launch_moe_combine(const JoinArgs &a, int type, hipStream_t s) { return launch_join(a, type, 1, s); }
hipError_t launch_moe_combine_grad(const JoinArgs &a, int type, hipStream_t s) { return launch_join(a, type, 2, s); }

}  // namespace spx
