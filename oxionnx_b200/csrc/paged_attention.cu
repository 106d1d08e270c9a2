// Causal attention of packed sequences' new rows over the pages of a cache: a warp for each row and head, one pass over the
// keys with the running maximum and sum of the softmax in f32.
#include "decoder_device.cuh"

namespace oxb {
namespace k {

namespace {

constexpr int kWarps = 8;

template <typename T>
__global__ void __launch_bounds__(kWarps * 32) paged_attention_rows(PagedAttention a) {
  pdl_enter();
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * kWarps + threadIdx.x / 32;
  if (row >= a.t.tokens * a.heads) return;
  const int token = (int)(row / a.heads), head = (int)(row % a.heads), kv = head / (a.heads / a.kv_heads);
  int b = 0;
  for (int base = 0; base < a.t.sequences; base += 32) b += __popc(__ballot_sync(0xffffffffu, base + lane < a.t.sequences && a.t.cu_query[base + lane + 1] <= token));
  int64_t last = -1;
  int wrong = 0;
  if (b < a.t.sequences) {
    bool bad;
    const Sequence q = sequence_of(a.t, b, &bad);
    if (bad || token < q.first || token >= q.first + q.rows) wrong = kErrLengths;
    else last = (int64_t)q.length - q.rows + (token - q.first);
    if (a.max_query > 0 && q.rows > a.max_query) wrong = kErrQueryLength;
  } else if (token < a.t.cu_query[a.t.sequences]) {
    wrong = kErrLengths;
  }
  float q[8], acc[8], most = -INFINITY, sum = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int d = lane + 32 * i;
    q[i] = d < a.size ? to_f32(((const T*)a.q)[row * a.size + d]) : 0.f;
    acc[i] = 0.f;
  }
  for (int64_t j = 0; j <= last; ++j) {
    const int page = a.t.page_table[(int64_t)b * a.t.max_pages + j / a.t.page];
    if (page < 0 || page >= a.t.pages) {
      wrong = kErrPage;
      continue;
    }
    const int64_t at = (((int64_t)page * a.t.page + j % a.t.page) * a.kv_heads + kv) * a.size;
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (lane + 32 * i < a.size) dot += q[i] * to_f32(((const T*)a.key_cache)[at + lane + 32 * i]);
    for (int o = 16; o > 0; o /= 2) dot += __shfl_xor_sync(0xffffffffu, dot, o);
    dot *= a.scale;
    const float next = fmaxf(most, dot);
    const float keep = most == -INFINITY ? 0.f : expf(most - next), p = expf(dot - next);
    most = next;
    sum = sum * keep + p;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (lane + 32 * i < a.size) acc[i] = acc[i] * keep + p * to_f32(((const T*)a.value_cache)[at + lane + 32 * i]);
  }
  if (wrong && lane == 0) report(a.err, wrong);
  const float scale = sum > 0.f ? 1.f / sum : 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (lane + 32 * i < a.size) ((T*)a.out)[row * a.size + lane + 32 * i] = from_f32<T>(last < 0 ? 0.f : acc[i] * scale);
}

}  // namespace

size_t paged_attention_workspace(const PagedAttention&) { return 0; }

void paged_attention(const PagedAttention& a, cudaStream_t s) {
  if (a.t.tokens == 0) return;
  const dim3 grid((unsigned)ceil_div(a.t.tokens * a.heads, kWarps));
  if (a.dt == DT::F16) launch(paged_attention_rows<__half>, grid, dim3(kWarps * 32), 0, s, a);
  else launch(paged_attention_rows<__nv_bfloat16>, grid, dim3(kWarps * 32), 0, s, a);
}

}  // namespace k
}  // namespace oxb
