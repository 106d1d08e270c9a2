// Device helpers that the decoder operators share.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "decoder.hpp"
#include "pdl.cuh"

namespace oxb {
namespace k {

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32(float v) { return __float2bfloat16_rn(v); }

// The new rows of sequence b, cut to the packed queries where the table runs past them, and its length, cut to what its row
// of the page table holds.  `bad` is set where anything had to be cut.
struct Sequence {
  int first, rows, length;
};
__device__ __forceinline__ Sequence sequence_of(const PagedTables& t, int b, bool* bad) {
  const int tokens = (int)t.tokens, a = t.cu_query[b], e = t.cu_query[b + 1], len = t.kv_lengths[b];
  const long long most = (long long)t.max_pages * t.page;
  const int first = min(max(a, 0), tokens), end = min(max(e, first), tokens), length = (int)min((long long)max(len, 0), most);
  *bad = first != a || end != e || length != len || (b == 0 && a != 0);
  return Sequence{first, end - first, length};
}

// The lowest nibbles of both halves of `w`, and `offset` beside them: a nibble in the low bits of a number whose last place is 1
// is 128 + code in bf16 and 1024 + code in f16.  One instruction; out of (w & mask) | constant the compiler made two, and the
// stream of 4096 x 65536 codes took 41.7 us in place of 36.8.
__device__ __forceinline__ uint32_t nibbles(uint32_t w, uint32_t offset) {
  uint32_t r;
  asm("lop3.b32 %0, %1, 0x000f000f, %2, 0xEA;" : "=r"(r) : "r"(w), "r"(offset));
  return r;
}
// A constant in a register, of which the compiler does not know that it is one.
__device__ __forceinline__ uint32_t in_register(uint32_t v) {
  uint32_t r;
  asm volatile("mov.b32 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

__device__ __forceinline__ void report(int* err, int code) { *(volatile int*)err = code; }

}  // namespace k
}  // namespace oxb
