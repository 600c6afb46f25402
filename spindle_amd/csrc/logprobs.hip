// Log probabilities of given tokens, entropy and the most likely alternatives of rows of logits
// (spx_logprobs).
//
// With x = logit / logit_scale, m = max x, S = sum exp(x - m) and T = sum (x - m) exp(x - m):
// log p_i = x_i - m - log S and the entropy is log S - T / S. One pass over the logits keeps m, S
// and T a lane (a larger maximum m' turns them into f S and f (T + (m - m') S), f = exp(m - m')) and
// the alternatives a wave: lane i holds the i-th best key. Bound by the bytes of the logits where
// there are many rows (500 rows of 151936 in fp32, one alternative: 66 us, 4.6 TB/s; twenty: 87), by the
// latency of two launches where there are few (one row: 6 us, with five alternatives 10). 72 rows of
// 49155 in 16 bits take 9 us, with twenty alternatives 20: the wave's first list is a sort by rank of its
// lanes' largest, later keys only those above the list's last.
#include "batch.h"
#include "dev.h"

namespace spx {

constexpr int LP_T = 256, LP_W = LP_T / 64;
constexpr float LOG2E = 1.4426950408889634f, LP_LOWEST = -3.402823466e38f, LP_FAR = -200.0f;

// Order of alternatives as one number: larger logit, then smaller id. 0: none.
__device__ __forceinline__ unsigned long long alt_key(float v, int id) {
  const uint32_t u = __float_as_uint(v);
  const uint32_t k = u & 0x80000000u ? ~u : u | 0x80000000u;
  return (unsigned long long)k << 32 | (uint32_t)~id;
}
__device__ __forceinline__ float alt_logit(unsigned long long key) {
  const uint32_t k = (uint32_t)(key >> 32);
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
__device__ __forceinline__ unsigned long long lane_u64(unsigned long long v, int src) {
  return (unsigned long long)(uint32_t)lane_i((int)(v >> 32), src) << 32 | (uint32_t)lane_i((int)(uint32_t)v, src);
}

// ------------------------------------------------------------------ the best keys of a wave
// Lane i holds the (i + 1)-th best key so far, 0 where there is none; `last` is the key that a
// better one has to beat (the top-th).
struct Best {
  unsigned long long mine, last;
  int top;
};
__device__ __forceinline__ void best_insert(Best &b, unsigned long long k) {  // k: the same in every lane
  const int lane = threadIdx.x & 63, pos = __builtin_popcountll(__builtin_amdgcn_ballot_w64(b.mine > k));
  const uint32_t hi = (uint32_t)__builtin_amdgcn_mov_dpp((int)(b.mine >> 32), 0x138, 0xF, 0xF, true);  // lane i - 1's (wave shift right)
  const uint32_t lo = (uint32_t)__builtin_amdgcn_mov_dpp((int)(uint32_t)b.mine, 0x138, 0xF, 0xF, true);
  const unsigned long long up = (unsigned long long)hi << 32 | lo;
  b.mine = lane < pos ? b.mine : lane == pos ? k : up;
  b.last = lane_u64(b.mine, b.top - 1);
}
// Every lane's key is offered.
__device__ __forceinline__ void best_offer(Best &b, unsigned long long key) {
  unsigned long long todo = __builtin_amdgcn_ballot_w64(key > b.last);
  while (todo) {
    const unsigned long long k = lane_u64(key, __builtin_ctzll(todo));
    todo &= todo - 1;
    if (k > b.last) best_insert(b, k);
  }
}
// The list from one key a lane (0: none): for few the largest one after the other, else each goes to the
// lane of its rank. Both ways, whole calls in us (one after the other / by rank):
//   top                    1            4            5            20
//   72 x 49155, bf16       12.9 / 16.2  15.5 / 16.3  16.5 / 16.4  30.9 / 19.1
//   1 x 151936, fp32       8.5 / 10.1   10.0 / 10.0  10.6 / 10.0  20.7 / 12.1
//   500 x 151936, fp32     66 / 69      71 / 72      73 / 73.5    104 / 87
__device__ __forceinline__ void best_start(Best &b, unsigned long long key, int top) {
  const int lane = threadIdx.x & 63;
  b.top = top;
  if (top <= 4) {
    b.mine = 0;
    for (int n = 0; n < top; n++) {
      const unsigned long long k = wave_max_u64(key);
      if (lane == n) b.mine = k;
      if (key == k) key = 0;
    }
  } else {
    if (key == 0) key = lane + 1;  // (numbers of their own, below every key)
    int rank = 0;
#pragma unroll
    for (int j = 0; j < 64; j++) rank += lane_u64(key, j) > key;
    const uint32_t hi = (uint32_t)__builtin_amdgcn_ds_permute(rank * 4, (int)(key >> 32)), lo = (uint32_t)__builtin_amdgcn_ds_permute(rank * 4, (int)(uint32_t)key);
    b.mine = hi ? (unsigned long long)hi << 32 | lo : 0ull;
  }
  b.last = lane_u64(b.mine, top - 1);
}

// ------------------------------------------------------------------ sums
struct Sums { float m, S, T; };
__device__ __forceinline__ void sums_join(Sums &a, const Sums &b) {
  // (differences below LP_FAR leave nothing: their exponential is 0; cut there, products stay finite)
  const float m = fmaxf(a.m, b.m), da = fmaxf(a.m - m, LP_FAR), db = fmaxf(b.m - m, LP_FAR);
  const float fa = __builtin_amdgcn_exp2f(da * LOG2E), fb = __builtin_amdgcn_exp2f(db * LOG2E);
  a.T = fa * fmaf(da, a.S, a.T) + fb * fmaf(db, b.S, b.T);
  a.S = fa * a.S + fb * b.S;
  a.m = m;
}
__device__ __forceinline__ Sums sums_from(const Sums &s, int x) {
  return {__shfl_xor(s.m, x), __shfl_xor(s.S, x), __shfl_xor(s.T, x)};
}
__device__ __forceinline__ void sums_wave(Sums &s) {
#pragma unroll
  for (int x = 1; x < 64; x <<= 1) sums_join(s, sums_from(s, x));
}

// ------------------------------------------------------------------ logits
template <int TYPE>
__device__ __forceinline__ float logit_one(const void *x, int64_t i, float lscale) {
  float v;
  if (TYPE == T_F32) v = ((const float *)x)[i];
  else if (TYPE == T_F16) v = (float)((const _Float16 *)x)[i];
  else v = __uint_as_float((uint32_t)((const uint16_t *)x)[i] << 16);
  return (lscale != 1.0f ? v / lscale : v) + 0.0f;  // (-0 becomes 0: the two are equal alternatives)
}
template <int TYPE, bool SCALED, int V>
__device__ __forceinline__ void logit_vec(uint4 r, float *v, float lscale) {
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int i = 0; i < V; i++) {
    if (TYPE == T_F32) v[i] = __uint_as_float(w[i]);
    else if (TYPE == T_F16) v[i] = h2f(w[i >> 1] >> (16 * (i & 1)));
    else v[i] = __uint_as_float(i & 1 ? w[i >> 1] & 0xffff0000u : w[i >> 1] << 16);
    v[i] = (SCALED ? v[i] / lscale : v[i]) + 0.0f;
  }
}

// N logits a lane, of ids id(0) .. id(N - 1), -inf where there is none. Ids of one call are larger
// than those of the wave's calls before, so that a value equal to the list's last one is no better.
template <int N, class F>
__device__ __forceinline__ void take(const float *v, F id, int top, bool &begun, Best &b, Sums &s) {
  float best = v[0];
#pragma unroll
  for (int i = 1; i < N; i++) best = fmaxf(best, v[i]);
  // one new maximum for the N: a NaN or +inf leaves S a NaN, -inf adds nothing
  const float m = fmaxf(s.m, best), d = fmaxf(s.m - m, LP_FAR), f = __builtin_amdgcn_exp2f(d * LOG2E);
  s.T = f * fmaf(d, s.S, s.T);
  s.S *= f;
  s.m = m;
#pragma unroll
  for (int i = 0; i < N; i++) {
    const float z = v[i] - m, e = __builtin_amdgcn_exp2f(z * LOG2E);
    s.S += e;
    s.T = fmaf(fmaxf(z, LP_FAR), e, s.T);
  }
  if (!top) return;
  auto key_of = [&](int i) { return v[i] > -__builtin_inff() ? alt_key(v[i], id(i)) : 0ull; };
  if (!begun) {
    begun = true;
    unsigned long long k = 0;
#pragma unroll
    for (int i = 0; i < N; i++) { const unsigned long long c = key_of(i); k = c > k ? c : k; }
    best_start(b, k, top);
    if (N > 1) {  // the others that may be among them (equal ones too: ids are in no order here)
      const float bar = b.last ? alt_logit(b.last) : -__builtin_inff();
#pragma unroll
      for (int i = 0; i < N; i++)
        if (__builtin_amdgcn_ballot_w64(v[i] >= bar)) {
          const unsigned long long c = key_of(i);
          best_offer(b, c == k ? 0ull : c);
        }
    }
  } else {
    const float bar = b.last ? alt_logit(b.last) : -__builtin_inff();
    if (__builtin_amdgcn_ballot_w64(best > bar)) {
#pragma unroll
      for (int i = 0; i < N; i++)
        if (__builtin_amdgcn_ballot_w64(v[i] > bar)) best_offer(b, key_of(i));
    }
  }
}

// A row's values, once its sums and its best keys are known (the latter in wave 0's lanes).
template <int TYPE>
__device__ __forceinline__ void finish(const LogprobArgs &a, int row, const Sums &s, unsigned long long key) {
  const int lane = threadIdx.x & 63;
  const bool bad = s.S != s.S, none = s.S == 0.0f;
  const float logS = logf(s.S), nan = __builtin_nanf("");
  if (lane == 0) {
    if (a.entropy) a.entropy[row] = bad ? nan : none ? 0.0f : logS - s.T / s.S;
    if (a.logp) {
      const int id = a.targets[row];
      float lp = nan;
      if (!bad && id >= 0 && id < a.vocab) {
        const float v = logit_one<TYPE>(a.x, (int64_t)row * a.ld + id, a.lscale);
        lp = v == -__builtin_inff() ? v : v - s.m - logS;
      }
      a.logp[row] = lp;
    }
  }
  if (lane < a.top) {
    const bool is = key != 0 && !bad;
    a.top_ids[(int64_t)row * a.top + lane] = is ? (int)~(uint32_t)key : -1;
    a.top_logp[(int64_t)row * a.top + lane] = bad ? nan : is ? alt_logit(key) - s.m - logS : -__builtin_inff();
  }
}

// The waves' sums and lists together, in wave 0: the first sixteen of each list are sorted at once, the
// others offered.
__device__ __forceinline__ void join_waves(Sums &s, Best &b, int top) {
  __shared__ Sums ss[LP_W];
  __shared__ unsigned long long sk[LP_W][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (lane == 0) ss[wave] = s;
  if (top) sk[wave][lane] = b.mine;
  __syncthreads();
  if (wave) return;
  for (int w = 1; w < LP_W; w++) sums_join(s, ss[w]);
  if (top) {
    const int w = lane >> 4, i = lane & 15;
    best_start(b, i < top ? sk[w][i] : 0ull, top);
    if (top > 16) best_offer(b, 16 + i < top ? sk[w][16 + i] : 0ull);
  }
}
static_assert(LP_W == 4, "a quarter of the wave a list");

// A workgroup takes a part of a row, its waves shares of that one after the other
// (ids ascend within a wave), 64 vectors of 16 bytes a load, four loads at a time. Elements before
// the first 16-byte boundary and behind the last one are one apiece for the first and last wave.
template <int TYPE, bool SCALED>
__global__ __launch_bounds__(LP_T) void k_logprobs(const LogprobArgs a, int parts) {
  constexpr int ES = TYPE == T_F32 ? 4 : 2, V = 16 / ES, U = 4;
  const int lane = threadIdx.x & 63, row = blockIdx.x / parts, part = blockIdx.x % parts;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const char *base = (const char *)a.x + (int64_t)row * a.ld * ES;
  const int head = min((int)((16 - ((uintptr_t)base & 15)) & 15) / ES, a.vocab), nvec = (a.vocab - head) / V, tail = a.vocab - head - nvec * V;
  const uint4 *vec = (const uint4 *)(base + head * ES);
  // 64 U vectors a turn, turns split evenly among all waves of the row
  const int turns = (nvec + 64 * U - 1) / (64 * U), waves = parts * LP_W, w = part * LP_W + wave;
  const int t0 = (int)((int64_t)turns * w / waves), t1 = (int)((int64_t)turns * (w + 1) / waves);
  Sums s{LP_LOWEST, 0.0f, 0.0f};
  Best b{0, 0, a.top};
  bool begun = false;
  if (w == 0 && head) {
    float v = lane < head ? logit_one<TYPE>(base, lane, a.lscale) : -__builtin_inff();
    take<1>(&v, [&](int) { return lane; }, a.top, begun, b, s);
  }
  for (int t = t0; t < t1; t++) {
    const int j = t * 64 * U + lane;
    float v[U * V];
#pragma unroll
    for (int u = 0; u < U; u++) {
      if (j + 64 * u < nvec) {
        logit_vec<TYPE, SCALED, V>(vec[j + 64 * u], v + u * V, a.lscale);
      } else {
#pragma unroll
        for (int i = 0; i < V; i++) v[u * V + i] = -__builtin_inff();
      }
    }
    take<U * V>(v, [&](int i) { return head + (j + 64 * (i / V)) * V + i % V; }, a.top, begun, b, s);
  }
  if (w == waves - 1 && tail) {
    const int i = head + nvec * V + lane;
    float v = lane < tail ? logit_one<TYPE>(base, i, a.lscale) : -__builtin_inff();
    take<1>(&v, [&](int) { return i; }, a.top, begun, b, s);
  }
  sums_wave(s);
  join_waves(s, b, a.top);
  if (wave) return;
  if (parts == 1) { finish<TYPE>(a, row, s, b.mine); return; }
  const int64_t at = (int64_t)row * parts + part;
  if (lane == 0) ((float4 *)a.ws)[at] = make_float4(s.m, s.S, s.T, 0.0f);
  // keys [row][place][part]: the best of every part come first
  if (lane < a.top) ((unsigned long long *)((float4 *)a.ws + (int64_t)a.rows * parts))[((int64_t)row * a.top + lane) * parts + part] = b.mine;
}

// The parts of a row together.
template <int TYPE>
__global__ __launch_bounds__(LP_T) void k_logprobs_join(const LogprobArgs a, int parts) {
  const int row = blockIdx.x, t = threadIdx.x;
  const float4 *sums = (const float4 *)a.ws + (int64_t)row * parts;
  const unsigned long long *keys = (const unsigned long long *)((const float4 *)a.ws + (int64_t)a.rows * parts) + (int64_t)row * a.top * parts;
  Sums s{LP_LOWEST, 0.0f, 0.0f};
  for (int p = t; p < parts; p += LP_T) {
    const float4 v = sums[p];
    sums_join(s, Sums{v.x, v.y, v.z});
  }
  sums_wave(s);
  Best b{0, 0, a.top};
  if (a.top) {
    best_start(b, t < parts * a.top ? keys[t] : 0ull, a.top);
    for (int p = LP_T; p < parts * a.top; p += LP_T) best_offer(b, p + t < parts * a.top ? keys[p + t] : 0ull);
  }
  join_waves(s, b, a.top);
  if (t < 64) finish<TYPE>(a, row, s, b.mine);
}

// Parts of a row: enough workgroups for two thousand (eight a CU), of 4096 logits at least: a turn a wave
// in fp32. (In 16 bits a turn is twice that, and half of the waves of parts that short have none.)
int logprobs_parts(int rows, int vocab) {
  const int most = (vocab + LP_W * 64 * 16 - 1) / (LP_W * 64 * 16);
  int parts = (2048 + rows - 1) / rows;
  return parts < most ? parts : most;
}

template <int TYPE>
static void launch_type(const LogprobArgs &a, int parts, hipStream_t s) {
  if (a.lscale != 1.0f) hipLaunchKernelGGL((k_logprobs<TYPE, true>), dim3(parts * a.rows), dim3(LP_T), 0, s, a, parts);
  else hipLaunchKernelGGL((k_logprobs<TYPE, false>), dim3(parts * a.rows), dim3(LP_T), 0, s, a, parts);
  if (parts > 1) hipLaunchKernelGGL(k_logprobs_join<TYPE>, dim3(a.rows), dim3(LP_T), 0, s, a, parts);
}

hipError_t launch_logprobs(const LogprobArgs &a, int type, hipStream_t s) {
  const int parts = logprobs_parts(a.rows, a.vocab);
  if (type == T_F32) launch_type<T_F32>(a, parts, s);
  else if (type == T_F16) launch_type<T_F16>(a, parts, s);
  else launch_type<T_BF16>(a, parts, s);
  return hipGetLastError();
}

}  // namespace spx
