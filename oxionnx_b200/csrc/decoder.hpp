// Launch interface of the decoder operators: 4-bit linears, the paged cache and the attention that reads it.  Host-callable,
// enqueues on a stream, never synchronises.
#pragma once

#include "common.hpp"

namespace oxb {
namespace k {

// Which pages hold which sequence.  Sequence b's new tokens are rows cu_query[b] .. cu_query[b+1] of the packed queries;
// with them it has kv_lengths[b] tokens, and token t lies in row t % page of page page_table[b][t / page].  A new row i of n
// has position kv_lengths[b] - n + i; a row of negative position belongs to nothing (an idle stream of a fixed batch): it is
// not appended and its results are 0, as are those of rows behind the last sequence.
struct PagedTables {
  const int* cu_query;    // [sequences + 1]
  const int* kv_lengths;  // [sequences]
  const int* page_table;  // [sequences][max_pages]
  int sequences, max_pages, page;
  int64_t pages;   // pages of the cache
  int64_t tokens;  // rows of the packed queries
};

// Codes of the error word (see error_text in runtime.cpp).
constexpr int kErrPage = 21, kErrPosition = 22, kErrLengths = 23, kErrQueryLength = 24;
constexpr int kMaxSequences = 4096;

struct PagedAppend {
  PagedTables t;
  const void *q, *k, *v;   // rows of the new tokens; a row starts q_stride (k_stride, v_stride) lanes behind the one before
  int64_t q_stride, k_stride, v_stride;
  void* rotated;           // [tokens][heads * size]
  void *key_cache, *value_cache;  // [pages][page][kv_heads][size]
  const float *cos, *sin;  // [positions][half], null without rotation
  int64_t positions;
  int heads, kv_heads, size, half;
  bool interleaved;
  DT in_dt, cache_dt;      // q / k / v: the cache's type or f32; rotated: the cache's type
  int* err;
};
void paged_append(const PagedAppend& a, cudaStream_t s);

struct PagedAttention {
  PagedTables t;
  const void* q;  // [tokens][heads * size]
  const void *key_cache, *value_cache;
  void* out;      // [tokens][heads * size]
  int heads, kv_heads, size;
  float scale;
  int max_query;  // most new rows of a sequence, 0: not known
  DT dt;
  void* workspace;  // of paged_attention_workspace bytes, zero before the first launch
  int* err;
};
size_t paged_attention_workspace(const PagedAttention& a);
void paged_attention(const PagedAttention& a, cudaStream_t s);
// Its sequences of at least `least_rows` packed rows (new rows times query heads of a key head), on tcgen05.
bool paged_attention_prompts_fit(const PagedAttention& a);
size_t paged_attention_prompts_workspace(const PagedAttention& a);
void paged_attention_prompts(const PagedAttention& a, int least_rows, void* workspace, cudaStream_t s);
int device_sms();

// y[m][n] = sum_k x[m][k] * (code[n][k] - zero[n][k / group]) * scale[n][k / group] + bias[n]
struct Linear4 {
  const void* x;
  void* y;
  const uint8_t* codes;
  const float* scales;
  const uint8_t* zeros;   // null: 8
  const float* bias;      // null: none
  int64_t rows;
  int k, n, group, groups;  // groups: of one output's inputs, the last one perhaps short
  DT dt;                    // x and y
};
void linear4(const Linear4& a, cudaStream_t s);

}  // namespace k
}  // namespace oxb
