// Block tables and slot maps of a step, built on the device from the sequences' lengths
// (spx_pages_plan).
//
// With l tokens held, a added and P tokens a page, a sequence lacks ceil((l + a) / P) - ceil(l / P)
// pages. Three running sums over the sequences place everything: pages that go back (where they
// land on the free list), pages lacked (which entries of the list a sequence takes, and whether
// they are there) and rows (where its rows start). Lacked pages are granted as long as the running
// sum stays within the list, so the granted sequences' shares lie without gaps from the list's end.
#include "batch.h"
#include "dev.h"

namespace spx {

constexpr int PLAN_T = 1024;
// Up to so many rows the one workgroup places the rows too (two a thread); beyond, a launch of their own
// is quicker than its turns: 21000 rows of 500 sequences 28 us in one launch, 14 us in two.
constexpr int PLAN_ROWS = 2048;

// Turns arr[0 .. n) into its running sum, arr[n] being the total, in place: arr[i] = sum of the
// values before i. Every thread of the workgroup calls it.
__device__ __forceinline__ void block_prefix(int *arr, int n, int *tmp) {
  const int t = threadIdx.x, wave = t >> 6, lane = t & 63;
  int carry = 0;
  for (int b = 0; b < n; b += PLAN_T) {
    const int i = b + t, v = i < n ? arr[i] : 0;
    const int up = wave_scan(v);
    if (lane == 63) tmp[wave] = up;
    __syncthreads();
    int before = carry, all = carry;
    for (int w = 0; w < PLAN_T / 64; w++) {
      const int x = tmp[w];
      if (w < wave) before += x;
      all += x;
    }
    if (i < n) arr[i] = before + up - v;
    carry = all;
    __syncthreads();
  }
  if (t == 0) arr[n] = carry;
  __syncthreads();
}

// The i with pre[i] <= k < pre[i + 1]; pre ascends, pre[0] = 0 <= k < pre[n].
__device__ __forceinline__ int find_share(const int *pre, int n, int k) {
  int lo = 0, hi = n;  // pre[lo] <= k < pre[hi]
  while (hi - lo > 1) {
    const int m = (lo + hi) >> 1;
    if (pre[m] <= k) lo = m; else hi = m;
  }
  return lo;
}

// One row's slot and position. Its sequence's new length and status say where its rows lie. (start:
// running sums of rows, which may end behind a.rows.)
__device__ __forceinline__ void plan_row(const PlanArgs &a, const int *start, int n, int r) {
  int slot = -1, pos = -1;
  if (r < start[n]) {
    const int s = find_share(start, n, r);
    if (a.status[s] == 0) {
      pos = a.lens_out[s] - (start[s + 1] - start[s]) + (r - start[s]);
      slot = (a.tables[(int64_t)s * a.cols + (pos >> a.page)] << a.page) + (pos & ((1 << a.page) - 1));
    }
  }
  a.slots[r] = slot;
  a.positions[r] = pos;
}

// One workgroup does it all but the rows of large steps, which k_pages_rows places: what it reads and writes
// is a few words a sequence, a page and a row, so a launch's latency and the dependent steps (read lengths,
// three scans, look up pages) bound it: 6.5 us for 24 sequences of a token each, 8.3 us
// for 500 with 21000 rows, 3.7 us more for the rows.
__global__ __launch_bounds__(PLAN_T) void k_pages_plan(const PlanArgs a) {
  __shared__ int back[PLAN_MAX_SEQ + 1], need[PLAN_MAX_SEQ + 1], start[PLAN_MAX_SEQ + 1], tmp[PLAN_T / 64];
  const int t = threadIdx.x, n = a.n_seq, P = 1 << a.page;
  // (a table may have room for more than 2^31 tokens, a length never: what is past it does not fit)
  const int64_t cap = min((int64_t)a.cols << a.page, (int64_t)INT32_MAX);
  const int had = min(max(a.n_free[0], 0), a.n_pages);
  auto held_of = [&](int s) { return (int)min((int64_t)max(a.lens[s], 0), cap); };
  for (int s = t; s < n; s += PLAN_T) {
    const int l = held_of(s), add = a.add[s], held = (int)(((int64_t)l + P - 1) >> a.page);
    const bool fits = add >= 0 && (int64_t)l + add <= cap;
    back[s] = add < 0 ? held : 0;
    need[s] = fits ? (int)(((int64_t)l + add + P - 1) >> a.page) - held : 0;
    start[s] = min(max(add, 0), a.rows + 1);  // (at most rows + 1 each: the running sum stays in 32 bits)
  }
  __syncthreads();
  block_prefix(back, n, tmp);
  block_prefix(start, n, tmp);
  // a sequence whose rows end behind the last one takes no pages
  for (int s = t; s < n; s += PLAN_T)
    if (start[s + 1] > a.rows) need[s] = 0;
  __syncthreads();
  block_prefix(need, n, tmp);
  const int freed = min(back[n], a.n_pages - had);  // (more than the list holds only from lengths that are not the pool's)
  for (int k = t; k < freed; k += PLAN_T) {
    const int s = find_share(back, n, k);
    a.free_list[had + k] = a.tables[(int64_t)s * a.cols + (k - back[s])];
  }
  const int avail = had + freed;
  __syncthreads();  // (the released pages are on the list, the lengths still as they came)
  int taken = 0;
  for (int s = t; s < n; s += PLAN_T) {
    const int l = held_of(s), add = a.add[s], mine = need[s + 1] - need[s];
    const bool ok = add >= 0 && (int64_t)l + add <= cap && start[s + 1] <= a.rows && (mine == 0 || need[s + 1] <= avail);
    if (ok && mine) taken = max(taken, need[s + 1]);
    a.status[s] = add >= 0 && !ok;
    a.lens_out[s] = add < 0 ? 0 : ok ? l + add : l;
  }
  // all granted shares together: the largest end among them
  taken = (int)wave_max_u32((uint32_t)taken);
  if ((t & 63) == 0) tmp[t >> 6] = taken;
  __syncthreads();
  for (int w = 0; w < PLAN_T / 64; w++) taken = max(taken, tmp[w]);
  for (int k = t; k < taken; k += PLAN_T) {
    const int s = find_share(need, n, k);
    const int total = a.lens_out[s], mine = need[s + 1] - need[s];  // granted: its length with the new rows
    const int first = (int)(((int64_t)total + P - 1) >> a.page) - mine;
    a.tables[(int64_t)s * a.cols + first + (k - need[s])] = a.free_list[avail - 1 - k];
  }
  for (int s = t; s <= n; s += PLAN_T) a.q_start[s] = min(start[s], a.rows);
  if (t == 0) a.n_free_out[0] = avail - taken;
  __syncthreads();
  if (a.rows <= PLAN_ROWS)
    for (int r = t; r < a.rows; r += PLAN_T) plan_row(a, start, n, r);
}

// The rows of a step of many, 256 a workgroup: each finds its sequence in q_start, which k_pages_plan
// left (a sequence that ends behind a.rows is cut there, and refused).
__global__ __launch_bounds__(256) void k_pages_rows(const PlanArgs a) {
  __shared__ int start[PLAN_MAX_SEQ + 1];
  for (int s = threadIdx.x; s <= a.n_seq; s += 256) start[s] = a.q_start[s];
  __syncthreads();
  const int r = blockIdx.x * 256 + threadIdx.x;
  if (r < a.rows) plan_row(a, start, a.n_seq, r);
}

hipError_t launch_pages_plan(const PlanArgs &a, hipStream_t s) {
  hipLaunchKernelGGL(k_pages_plan, dim3(1), dim3(PLAN_T), 0, s, a);
  if (a.rows > PLAN_ROWS) hipLaunchKernelGGL(k_pages_rows, dim3((a.rows + 255) / 256), dim3(256), 0, s, a);
  return hipGetLastError();
}

}  // namespace spx
