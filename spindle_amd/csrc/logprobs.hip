// Log probabilities of given tokens, entropy and the most likely alternatives of rows of logits
// (spx_logprobs).
//
// With x = logit / logit_scale, m = max x, S = sum exp(x - m) and T = sum (x - m) exp(x - m):
// log p_i = x_i - m - log S and the entropy is log S - T / S.
#include "batch.h"
#include "dev.h"

namespace spx {

constexpr int LP_T = 1024;

template <int TYPE>
__device__ __forceinline__ float logit_at(const void *x, int64_t i, float lscale) {
  float v;
  if (TYPE == T_F32) v = ((const float *)x)[i];
  else if (TYPE == T_F16) v = (float)((const _Float16 *)x)[i];
  else v = __uint_as_float((uint32_t)((const uint16_t *)x)[i] << 16);
  return (lscale != 1.0f ? v / lscale : v) + 0.0f;  // (-0 becomes 0: the two are equal alternatives)
}
// Order of alternatives as one number: larger logit, then smaller id. Never 0.
__device__ __forceinline__ unsigned long long alt_key(float v, int id) {
  const uint32_t u = __float_as_uint(v);
  const uint32_t k = u & 0x80000000u ? ~u : u | 0x80000000u;
  return (unsigned long long)k << 32 | (uint32_t)~id;
}
__device__ __forceinline__ float alt_logit(unsigned long long key) {
  const uint32_t k = (uint32_t)(key >> 32);
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

template <int TYPE>
__global__ __launch_bounds__(LP_T) void k_logprobs(const LogprobArgs a) {
  __shared__ float red[LP_T / 64][2];
  __shared__ unsigned long long best[LP_T / 64];
  const int t = threadIdx.x, wave = t >> 6, lane = t & 63, row = blockIdx.x;
  const int64_t at = (int64_t)row * a.ld;
  float m = -__builtin_inff();
  bool bad = false;
  for (int i = t; i < a.vocab; i += LP_T) {
    const float v = logit_at<TYPE>(a.x, at + i, a.lscale);
    bad |= !(v < __builtin_inff());
    m = fmaxf(m, v);
  }
  bad = __syncthreads_or(bad);
  m = wave_max(m);
  if (lane == 0) red[wave][0] = m;
  __syncthreads();
  for (int w = 0; w < LP_T / 64; w++) m = fmaxf(m, red[w][0]);
  __syncthreads();
  const bool none = m == -__builtin_inff();
  float S = 0.0f, T = 0.0f;
  if (!bad && !none)
    for (int i = t; i < a.vocab; i += LP_T) {
      const float z = fmaxf(logit_at<TYPE>(a.x, at + i, a.lscale) - m, -200.0f), e = expf(z);
      S += e;
      T = fmaf(z, e, T);
    }
  S = wave_sum(S);
  T = wave_sum(T);
  if (lane == 0) { red[wave][0] = S; red[wave][1] = T; }
  __syncthreads();
  S = T = 0.0f;
  for (int w = 0; w < LP_T / 64; w++) { S += red[w][0]; T += red[w][1]; }
  const float logS = logf(S);
  if (t == 0) {
    if (a.entropy) a.entropy[row] = bad ? __builtin_nanf("") : none ? 0.0f : logS - T / S;
    if (a.logp) {
      float lp = __builtin_nanf("");
      const int id = a.targets[row];
      if (!bad && id >= 0 && id < a.vocab) {
        const float v = logit_at<TYPE>(a.x, at + id, a.lscale);
        lp = v == -__builtin_inff() ? v : v - m - logS;
      }
      a.logp[row] = lp;
    }
  }
  unsigned long long last = ~0ull;
  for (int n = 0; n < a.top; n++) {
    unsigned long long k = 0;
    if (!bad && last)
      for (int i = t; i < a.vocab; i += LP_T) {
        const float v = logit_at<TYPE>(a.x, at + i, a.lscale);
        const unsigned long long c = v == -__builtin_inff() ? 0ull : alt_key(v, i);
        if (c < last && c > k) k = c;
      }
    k = wave_max_u64(k);
    if (lane == 0) best[wave] = k;
    __syncthreads();
    for (int w = 0; w < LP_T / 64; w++) k = best[w] > k ? best[w] : k;
    __syncthreads();
    last = k;
    if (t == 0) {
      a.top_ids[(int64_t)row * a.top + n] = k ? (int)~(uint32_t)k : -1;
      a.top_logp[(int64_t)row * a.top + n] = bad ? __builtin_nanf("") : k ? alt_logit(k) - m - logS : -__builtin_inff();
    }
  }
}

hipError_t launch_logprobs(const LogprobArgs &a, int type, hipStream_t s) {
  if (type == T_F32) hipLaunchKernelGGL(k_logprobs<T_F32>, dim3(a.rows), dim3(LP_T), 0, s, a);
  else if (type == T_F16) hipLaunchKernelGGL(k_logprobs<T_F16>, dim3(a.rows), dim3(LP_T), 0, s, a);
  else hipLaunchKernelGGL(k_logprobs<T_BF16>, dim3(a.rows), dim3(LP_T), 0, s, a);
  return hipGetLastError();
}

}  // namespace spx
