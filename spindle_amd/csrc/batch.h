// Operators for batches of sequences: page planning (pages.hip), the paged 4-bit cache and
// attention over it (kv4.hip), log probabilities (logprobs.hip). Their C entries, with the checks
// of arguments, are in batch.cpp.
#pragma once
#include "../../include/spx.h"
#include "common.h"

namespace spx {

constexpr int PLAN_MAX_SEQ = 4096;

struct PlanArgs {
  int n_seq, page, cols, n_pages, rows;  // page: log2 of a page's tokens
  const int32_t *lens, *add, *n_free;
  int32_t *tables, *free_list, *lens_out, *n_free_out, *q_start, *slots, *positions, *status;
};
hipError_t launch_pages_plan(const PlanArgs &a, hipStream_t s);

struct Kv4Rows {  // append: k, v are read; read: written
  uint8_t *pool;
  int n_kv, page, n_pages, rows;  // page: log2 of a page's tokens
  void *k, *v;
  int64_t ld_k, ld_v;
  const int32_t *slots;
};
hipError_t launch_kv4_append(const Kv4Rows &a, int hd, int type, hipStream_t s);
hipError_t launch_kv4_read(const Kv4Rows &a, int hd, int type, hipStream_t s);

struct Kv4Attn {
  const uint8_t *pool;
  int n_kv, page, n_pages;  // page: log2 of a page's tokens
  const void *q;
  void *out;
  int64_t ld_q, ld_out;
  int group, rows, n_seq, cols, window;
  const int32_t *q_start, *kv_lens, *tables;
  float scale;  // times log2(e)
  int qvec, ovec;     // queries / outputs lie at multiples of 16 bytes
  int few;            // sequences with more rows (new tokens x query heads a key head) are k_kv4_rows'
  int chunk, rchunk;  // tokens a workgroup takes at a time
  float *part, *rpart;  // scratch: outputs, then (maximum, sum), of every job, key head, split and row
};
int64_t kv4_attention_ws(int hd, int group, int n_kv, int rows, int n_seq, int max_kv);
hipError_t launch_kv4_attention(Kv4Attn a, int hd, int type, int max_kv, hipStream_t s);

struct LogprobArgs {
  const void *x;
  int64_t ld;
  int rows, vocab, top;
  float lscale;
  const int32_t *targets;
  float *logp, *entropy, *top_logp;
  int32_t *top_ids;
  void *ws;
};
int logprobs_parts(int rows, int vocab);
hipError_t launch_logprobs(const LogprobArgs &a, int type, hipStream_t s);

}  // namespace spx
