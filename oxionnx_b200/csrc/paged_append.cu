// New tokens into a paged cache: queries and keys are rotated by their positions, keys and values go to their rows of the
// pages.  Memory bound: every lane is read once and written once, and a pair (a, b) of lanes at position p becomes
// (a cos - b sin, b cos + a sin) with the row p of cos and sin, in f32, rounded once.  64 tokens of 32 + 2 x 8 heads of 128 take
// 3.3 us, a launch and two dependent rounds of loads; 8100 of 16 + 2 x 16 heads of 64 take 24.8, 4.0 TB/s.
#include "decoder_device.cuh"

namespace oxb {
namespace k {

namespace {

constexpr int kAppendThreads = 256;

enum class Turn { None, Halves, Pairs, Lanes };  // pairs a half apart / side by side, in 16-byte steps; lane by lane

template <typename T>
struct alignas(16) Eight {
  T v[8];
};

template <typename TI>
__device__ __forceinline__ void load8(const TI* p, float* x) {
  if constexpr (sizeof(TI) == 4) {
    const float4 a = *(const float4*)p, b = *(const float4*)(p + 4);
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
  } else {
    const Eight<TI> r = *(const Eight<TI>*)p;
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = to_f32(r.v[i]);
  }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float* x) {
  Eight<T> r;
#pragma unroll
  for (int i = 0; i < 8; ++i) r.v[i] = from_f32<T>(x[i]);
  *(Eight<T>*)p = r;
}

// Where a token's lanes go: position -1 and slot -1 for a token of no sequence, slot -1 for one that something is wrong with.
struct Place {
  int64_t position, slot;
};
// `b`: the token's sequence, as many of the row bounds behind the first as lie at or before it.
__device__ __forceinline__ Place place_of(const PagedAppend& a, int64_t token, int b, int* wrong) {
  Place p{-1, -1};
  if (b < a.t.sequences) {
    bool bad;
    const Sequence q = sequence_of(a.t, b, &bad);
    if (bad || token < q.first || token >= q.first + q.rows) {
      *wrong = kErrLengths;
    } else {
      p.position = (int64_t)q.length - q.rows + (token - q.first);
      if (p.position >= 0) {
        const int position = (int)p.position, page = a.t.page_table[(int64_t)b * a.t.max_pages + position / a.t.page];
        if (a.cos && position >= a.positions) *wrong = kErrPosition;
        else if (page < 0 || page >= a.t.pages) *wrong = kErrPage;
        else p.slot = (int64_t)page * a.t.page + position % a.t.page;
      }
    }
  } else if (token < a.t.cu_query[a.t.sequences]) {
    *wrong = kErrLengths;  // bounds that fall
  }
  return p;
}

// An item is the 16 bytes of one head that a thread takes, or with Turn::Halves the two times 16 bytes whose lanes turn
// together.  Heads of q, then of k, then of v.
template <typename TI, typename T, Turn TURN>
struct Item {
  int h, lane;
  bool is_q, is_v, turns, two;

  __device__ __forceinline__ void locate(const PagedAppend& a, int item, int items_rotated, int items_plain) {
    const int turned = (a.heads + a.kv_heads) * items_rotated;
    int head, at;
    if (item < turned) head = item / items_rotated, at = item % items_rotated;
    else head = a.heads + a.kv_heads + (item - turned) / items_plain, at = (item - turned) % items_plain;
    is_q = head < a.heads, is_v = head >= a.heads + a.kv_heads;
    h = is_q ? head : is_v ? head - a.heads - a.kv_heads : head - a.heads;
    lane = at * 8;  // in the head
    turns = TURN != Turn::None && !is_v, two = false;
    if (TURN == Turn::Halves && turns) {
      two = at < a.half / 8;
      if (!two) lane = 2 * a.half + (at - a.half / 8) * 8, turns = false;
    } else if (turns) {
      turns = lane < 2 * a.half;
    }
  }
  __device__ __forceinline__ const TI* source(const PagedAppend& a, int64_t token) const {
    return (is_q ? (const TI*)a.q + token * a.q_stride : is_v ? (const TI*)a.v + token * a.v_stride : (const TI*)a.k + token * a.k_stride) + h * a.size;
  }
  __device__ __forceinline__ void fetch(const PagedAppend& a, int64_t token, float (&x)[8], float (&y)[8]) const {
    const TI* const src = source(a, token);
    load8(src + lane, x);
    if (two) load8(src + lane + a.half, y);
  }
  __device__ __forceinline__ void put(const PagedAppend& a, int64_t token, Place p, float (&x)[8], float (&y)[8]) const {
    if (p.slot < 0 && !is_q) return;
    T* dst = is_q ? (T*)a.rotated + (token * a.heads + h) * a.size : (is_v ? (T*)a.value_cache : (T*)a.key_cache) + (p.slot * a.kv_heads + h) * a.size;
    if (p.slot < 0) {  // a token of no sequence
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = y[i] = 0.f;
    } else if (turns) {
      const float *cos = a.cos + p.position * a.half, *sin = a.sin + p.position * a.half;
      if constexpr (TURN == Turn::Halves) {
        float c[8], s[8];
        load8(cos + lane, c);
        load8(sin + lane, s);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float u = x[i], v = y[i];
          x[i] = u * c[i] - v * s[i];
          y[i] = v * c[i] + u * s[i];
        }
      } else if constexpr (TURN == Turn::Pairs) {
        const float4 c = *(const float4*)(cos + lane / 2), s = *(const float4*)(sin + lane / 2);
        const float cc[4] = {c.x, c.y, c.z, c.w}, ss[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float u = x[2 * i], v = x[2 * i + 1];
          x[2 * i] = u * cc[i] - v * ss[i];
          x[2 * i + 1] = v * cc[i] + u * ss[i];
        }
      } else if constexpr (TURN == Turn::Lanes) {
        for (int i = 0; i < 8; ++i) {
          const int l = lane + i;
          if (l >= 2 * a.half) break;
          const bool second = a.interleaved ? l & 1 : l >= a.half;
          const int other = a.interleaved ? l ^ 1 : second ? l - a.half : l + a.half, turn = a.interleaved ? l / 2 : second ? l - a.half : l;
          const float w = to_f32(source(a, token)[other]);
          x[i] = second ? x[i] * cos[turn] + w * sin[turn] : x[i] * cos[turn] - w * sin[turn];
        }
      }
    }
    store8(dst + lane, x);
    if (two) store8(dst + lane + a.half, y);
  }
};

// A few tokens: a block serves one of them, or a part of its heads; its lanes are on their way while it looks where they go.
template <typename TI, typename T, Turn TURN>
__global__ void __launch_bounds__(kAppendThreads) paged_append_few(PagedAppend a, int parts, int items_rotated, int items_plain) {
  pdl_enter();
  const int64_t token = blockIdx.x / parts;
  const int item = (int)(blockIdx.x % parts) * kAppendThreads + threadIdx.x;
  const bool mine = item < (a.heads + a.kv_heads) * items_rotated + a.kv_heads * items_plain;
  Item<TI, T, TURN> it;
  float x[8], y[8];
  if (mine) {
    it.locate(a, item, items_rotated, items_plain);
    it.fetch(a, token, x, y);
  }
  int b = 0;
  for (int base = 0; base < a.t.sequences; base += 32) {
    const int i = base + (threadIdx.x & 31);
    b += __popc(__ballot_sync(0xffffffffu, i < a.t.sequences && a.t.cu_query[i + 1] <= token));
  }
  int wrong = 0;
  const Place p = place_of(a, token, b, &wrong);
  if (wrong && threadIdx.x == 0) report(a.err, wrong);
  if (mine) it.put(a, token, p, x, y);
}

// Many tokens: a thread takes the same item of kTokens of them, so that finding out which it is costs once: 8100 tokens of 48
// heads of 64 lanes 24.8 us (4.1 TB/s of what must move; 4 and 16 tokens 26.9, a block for each token 54, items out of one
// sequence of numbers with a division each 43).  Two tokens in flight cost 25.6: the registers are worth more as warps.
constexpr int kTokens = 8, kManyThreads = 512;
template <typename TI, typename T, Turn TURN>
__global__ void __launch_bounds__(kManyThreads) paged_append_many(PagedAppend a, int parts, int items_rotated, int items_plain) {
  __shared__ Place places[kTokens];
  pdl_enter();
  const int64_t token0 = (int64_t)(blockIdx.x / parts) * kTokens;
  const int tokens = (int)min((int64_t)kTokens, a.t.tokens - token0), warp = threadIdx.x / 32, lane = threadIdx.x & 31;
  const int item = (int)(blockIdx.x % parts) * blockDim.x + threadIdx.x;
  const bool mine = item < (a.heads + a.kv_heads) * items_rotated + a.kv_heads * items_plain;
  Item<TI, T, TURN> it;
  it.locate(a, mine ? item : 0, items_rotated, items_plain);
  for (int e = warp; e < tokens; e += blockDim.x / 32) {  // a warp looks a token up
    int b = 0;
    for (int base = 0; base < a.t.sequences; base += 32) b += __popc(__ballot_sync(0xffffffffu, base + lane < a.t.sequences && a.t.cu_query[base + lane + 1] <= token0 + e));
    if (lane == 0) {
      int wrong = 0;
      places[e] = place_of(a, token0 + e, b, &wrong);
      if (wrong) report(a.err, wrong);
    }
  }
  __syncthreads();
  if (!mine) return;
  for (int e = 0; e < tokens; ++e) {
    float x[8], y[8];
    it.fetch(a, token0 + e, x, y);
    it.put(a, token0 + e, places[e], x, y);
  }
}

template <typename TI, typename T>
void append_typed(const PagedAppend& a, cudaStream_t s) {
  Turn turn = Turn::None;
  if (a.cos) turn = a.interleaved ? (a.half % 4 == 0 ? Turn::Pairs : Turn::Lanes) : (a.half % 8 == 0 ? Turn::Halves : Turn::Lanes);
  const int plain = a.size / 8, rotated = turn == Turn::Halves ? plain - a.half / 8 : plain;
  const int items = (a.heads + a.kv_heads) * rotated + a.kv_heads * plain, parts = (int)ceil_div(items, kAppendThreads);
  const int many_parts = (int)ceil_div(items, kManyThreads), many_threads = (int)align_up((size_t)ceil_div(items, many_parts), 32);
  auto few = [&](auto kernel) { launch(kernel, dim3((unsigned)(a.t.tokens * parts)), dim3(kAppendThreads), 0, s, a, parts, rotated, plain); };
  auto many = [&](auto kernel) { launch(kernel, dim3((unsigned)(ceil_div(a.t.tokens, kTokens) * many_parts)), dim3(many_threads), 0, s, a, many_parts, rotated, plain); };
  const bool lot = a.t.tokens >= 148 * kTokens;  // blocks for each SM
  switch (turn) {
    case Turn::None: return lot ? many(paged_append_many<TI, T, Turn::None>) : few(paged_append_few<TI, T, Turn::None>);
    case Turn::Halves: return lot ? many(paged_append_many<TI, T, Turn::Halves>) : few(paged_append_few<TI, T, Turn::Halves>);
    case Turn::Pairs: return lot ? many(paged_append_many<TI, T, Turn::Pairs>) : few(paged_append_few<TI, T, Turn::Pairs>);
    case Turn::Lanes: return lot ? many(paged_append_many<TI, T, Turn::Lanes>) : few(paged_append_few<TI, T, Turn::Lanes>);
  }
}

}  // namespace

void paged_append(const PagedAppend& a, cudaStream_t s) {
  if (a.t.tokens == 0) return;
  const bool f32 = a.in_dt == DT::F32;
  if (a.cache_dt == DT::F16) f32 ? append_typed<float, __half>(a, s) : append_typed<__half, __half>(a, s);
  else f32 ? append_typed<float, __nv_bfloat16>(a, s) : append_typed<__nv_bfloat16, __nv_bfloat16>(a, s);
}

}  // namespace k
}  // namespace oxb
