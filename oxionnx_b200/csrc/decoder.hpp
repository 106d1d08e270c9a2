// Launch interface of the decoder operators: 4-bit linears, the paged cache and the attention that reads it.  Host-callable,
// enqueues on a stream, never synchronises.
#pragma once

#include <vector>

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

// Codes of the error word (see error_text in runtime.cpp), none of which a wait of another kernel has.
constexpr int kErrPage = 71, kErrPosition = 72, kErrLengths = 73, kErrQueryLength = 74;
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
  // laid out as Linear4Layout has them
  const void* codes;
  const void* scales;
  const uint8_t* zeros;   // null: 8
  bool scales_f16;        // scales are f16, f32 otherwise
  const float* unfold;    // [n]: what the sums of an output are multiplied by, powers of two; null: nothing
  bool exact_weights;     // 16-bit rows: their weights may not be rounded, however many rows there are
  const float* bias;      // null: none
  int64_t rows;
  int k, n, group, groups;  // groups: of one output's inputs, the last one perhaps short
  DT dt;                    // x and y
  void* workspace;          // linear4_workspace bytes, or null
  int* err;
};
// Powers of two by which each output's scales [n][groups] are multiplied before the weights are rounded to x's type, so that none
// overflows or loses bits (empty: all 0).  False where there are none, and the weights must not be rounded.
bool linear4_folds(const Linear4& a, const float* scales, bool zero_points, std::vector<int>* folds);
size_t linear4_workspace(const Linear4& a);
void linear4(const Linear4& a, cudaStream_t s);
bool linear4_many_rows(const Linear4& a);
void linear4_prompt(const Linear4& a, cudaStream_t s);  // many rows of 16 bits

// Where codes, scales and zero points of an [n][k] matrix lie on the device.  Outputs come in tiles of 16 (the last ones filled
// up with outputs of scale 0), inputs in blocks of 64 (filled up with any code: x is 0 there).  A block of a tile is 512 bytes,
// 16 for each lane of a warp: lane (g, q) = (lane / 4, lane % 4) has four inputs of every 16, 4 q on, of the outputs g and g + 8;
// a word holds those of 32 inputs, the even ones in nibbles 0-3 and the odd ones in 4-7.  So a group of 16 is one fragment's.  Scales and zero points (a byte each) of a tile
// and a group lie side by side, output g at 2 g and output g + 8 at 2 g + 1.
struct Linear4Layout {
  static int64_t tiles(int64_t n) { return (n + 63) / 64 * 4; }  // whole runs of four: no kernel has to look where they end
  static int64_t code_bytes(int64_t n, int64_t k) { return tiles(n) * ((k + 63) / 64) * 512; }
  static int64_t of_group(int64_t n, int64_t group, int64_t groups) { return (n / 16 * groups + group) * 16 + n % 8 * 2 + n % 16 / 8; }
  // packed[n][groups][group / 2]: two codes a byte, the even one low
  static void codes(const float* packed, int64_t n, int64_t k, int64_t group, uint8_t* out) {
    const int64_t blocks = (k + 63) / 64, row_bytes = (k + group - 1) / group * (group / 2);
    uint32_t* const words = (uint32_t*)out;
    for (int64_t o = 0; o < n; ++o)
      for (int64_t w = 0; w < blocks * 8; ++w) {  // word (w % 2) of lane q = w / 2 % 4 in block w / 8
        const int64_t q = w / 2 % 4;
        uint32_t v = 0;
        for (int64_t j = 0; j < 4; ++j) {  // two inputs each
          const int64_t at = w / 8 * 32 + w % 2 * 16 + j / 2 * 8 + q * 2 + j % 2;
          const uint32_t byte = at < row_bytes ? (uint32_t)packed[o * row_bytes + at] : 0u;
          v |= (byte & 15u) << (4 * j) | (byte >> 4) << (16 + 4 * j);
        }
        words[((o / 16 * blocks + w / 8) * 32 + o % 8 * 4 + q) * 4 + o % 16 / 8 * 2 + w % 2] = v;
      }
  }
};

}  // namespace k
}  // namespace oxb
