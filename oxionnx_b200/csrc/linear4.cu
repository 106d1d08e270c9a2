// Rows times a matrix of 4-bit codes with a scale (and a zero point) for each group of inputs,
//   y[m][n] = sum over groups g of scale[n][g] * sum over k in g of x[m][k] (code[n][k] - zero[n][g])  + bias[n],
// for few rows: what bounds it is reading the codes once.
//
// The codes are laid out once, when a session is planned, in the order in which the lanes of a warp take them (Linear4Layout):
// 16 bytes a lane are the m16n8k16 fragments of 16 outputs by 64 inputs.  Outputs are the fragments' rows and x's rows their
// columns, so that up to 8 rows cost no more instructions than one.  code - zero is a whole number below 16 in size and exact
// in either 16-bit type, so the products are exact and the sums are f32; a group's sum is scaled in f32.  f32 rows are taken
// as the sum of three bf16 numbers (8 bits of the significand each, all 24 of them, cut off and not rounded, so that the largest
// numbers stay finite), whose products are exact as well.
//
// A block has 16, 32 or 64 outputs and splits the inputs over its warps; the warps' sums meet in shared memory in one order.
// Rows that fit shared memory over many inputs have a kernel of their own, whose blocks stay (linear4_stream): 1 x 4096 x 16384
// takes 10.0 us in place of 11.5, 1 x 4096 x 65536 30, 4.6 TB/s.  What bounds both is the decoding, about 80 instructions for 16
// outputs by 64 inputs, of which 28 run on the pipe of shifts and logic at half rate.
#include <cooperative_groups.h>

#include <algorithm>
#include <mutex>
#include <type_traits>

#include "decoder_device.cuh"

namespace oxb {
namespace k {

namespace {

namespace cg = cooperative_groups;

constexpr int kWarps = 8;

template <typename T>
struct Operand {  // what the tensor cores multiply
  using type = T;
};
template <>
struct Operand<float> {
  using type = __nv_bfloat16;
};

template <typename H>
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Where `nibbles` puts them: into 128 in bf16, 1024 in f16.
template <typename H>
constexpr uint32_t kOffset = 0;
template <>
constexpr uint32_t kOffset<__half> = 0x64006400u;
template <>
constexpr uint32_t kOffset<__nv_bfloat16> = 0x43004300u;

template <typename H>
__device__ __forceinline__ uint32_t minus(uint32_t a, uint32_t b);
template <>
__device__ __forceinline__ uint32_t minus<__half>(uint32_t a, uint32_t b) {
  const __half2 r = __hsub2(*(const __half2*)&a, *(const __half2*)&b);
  return *(const uint32_t*)&r;
}
template <>
__device__ __forceinline__ uint32_t minus<__nv_bfloat16>(uint32_t a, uint32_t b) {
  const __nv_bfloat162 r = __hsub2(*(const __nv_bfloat162*)&a, *(const __nv_bfloat162*)&b);
  return *(const uint32_t*)&r;
}

// Four lanes of x from `src` (those from `left` on are zeros) as `SPLIT` numbers each, two to a word.
template <typename T, int SPLIT>
__device__ __forceinline__ void load4(const T* src, int left, bool whole, uint32_t (&w)[SPLIT][8], int at) {
  if constexpr (sizeof(T) == 2) {
    if (whole) {
      const uint2 a = *(const uint2*)src;
      w[0][at] = a.x, w[0][at + 1] = a.y;
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t lo = 2 * i < left ? *(const uint16_t*)(src + 2 * i) : 0u, hi = 2 * i + 1 < left ? *(const uint16_t*)(src + 2 * i + 1) : 0u;
        w[0][at + i] = lo | hi << 16;
      }
    }
  } else {
    float v[4];
    if (whole) {
      *(float4*)v = *(const float4*)src;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = i < left ? src[i] : 0.f;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float a = v[2 * i], b = v[2 * i + 1];
#pragma unroll
      for (int s = 0; s < SPLIT; ++s) {
        w[s][at + i] = __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x7632);  // the upper halves: 8 bits of the significand, cut off
        // an infinity's remainder is 0, not infinity minus infinity
        a = fabsf(a) == INFINITY ? 0.f : a - __uint_as_float(__float_as_uint(a) & 0xffff0000u);
        b = fabsf(b) == INFINITY ? 0.f : b - __uint_as_float(__float_as_uint(b) & 0xffff0000u);
      }
    }
  }
}

// MT: tiles of 16 outputs; NT: of 8 rows; SUB: groups of a 64-input block (4, 2 or 1); ZP: zero points, 8 without; ST: type of
// the scales.  `shift`: log2 of the blocks of a group where a group is at least a block.  The blocks of a cluster split the
// inputs further.
template <typename T, int MT, int NT, int SUB, bool ZP, typename ST>
__global__ void __launch_bounds__(kWarps * 32) linear4_rows(Linear4 a, int64_t row0, int shift, int splits) {
  using H = typename Operand<T>::type;
  constexpr int SPLIT = sizeof(T) == 4 ? 3 : 1, STEPS = 4 / SUB;  // k16 steps of a group within the block
  constexpr int LD = NT * 8 + 1;
  __shared__ float meet[kWarps / 2][MT * 16][LD], sums[MT * 16 * NT * 8];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  const int tile0 = blockIdx.x / splits * MT, slice = blockIdx.x % splits * kWarps + warp, blocks = (a.k + 63) / 64;
  row0 += (int64_t)blockIdx.y * NT * 8;
  const uint32_t offset = in_register(kOffset<H>);
  const int first = (int)((int64_t)blocks * slice / (splits * kWarps)), last = (int)((int64_t)blocks * (slice + 1) / (splits * kWarps));
  const int rows = (int)min((int64_t)NT * 8, a.rows - row0);
  const bool aligned = a.k % 4 == 0 && ((uintptr_t)a.x & 15) == 0;

  // addresses: one for the thread block and 32 bits for the lane (the layout fills the last blocks' tiles up)
  const uint8_t* const codes = (const uint8_t*)a.codes + (int64_t)tile0 * blocks * 512;
  const uint8_t* const scales = (const uint8_t*)a.scales + (int64_t)tile0 * a.groups * 16 * sizeof(ST);
  const uint8_t* const zeros = ZP ? a.zeros + (int64_t)tile0 * a.groups * 16 : nullptr;
  const T* const x_base = (const T*)a.x + row0 * a.k;
  const uint32_t lane_codes = lane * 16;
  uint32_t x_at[NT];  // rows behind the last are copies of it: their columns of the products go nowhere
#pragma unroll
  for (int t = 0; t < NT; ++t) x_at[t] = (uint32_t)min(t * 8 + g, rows - 1) * a.k + q * 4;

  float acc[MT][NT][4] = {};
  // the codes are the session's own: the first of them need not wait for the kernel in front
  uint4 ahead[MT];
  if (first < last)
#pragma unroll
    for (int m = 0; m < MT; ++m) ahead[m] = __ldcs((const uint4*)(codes + (uint32_t)(m * blocks + first) * 512u + lane_codes));
  asm volatile("griddepcontrol.wait;" ::: "memory");

#pragma unroll 2
  for (int b = first; b < last; ++b) {
    uint32_t x[NT][SPLIT][8];
    if (aligned && b * 64 + 64 <= a.k) {
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j) load4<T, SPLIT>(x_base + (x_at[t] + (uint32_t)(b * 64 + j * 16)), 4, true, x[t], 2 * j);
    } else {
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j) load4<T, SPLIT>(x_base + (x_at[t] + (uint32_t)(b * 64 + j * 16)), a.k - (b * 64 + j * 16 + q * 4), false, x[t], 2 * j);
    }
    uint4 w[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      w[m] = ahead[m];
      if (b + 1 < last) ahead[m] = __ldcs((const uint4*)(codes + (uint32_t)(m * blocks + b + 1) * 512u + lane_codes));
    }
#pragma unroll
    for (int m = 0; m < MT; ++m) {
#pragma unroll
      for (int s = 0; s < SUB; ++s) {
        const int group = SUB == 1 ? b >> shift : min(b * SUB + s, a.groups - 1);  // a block's groups behind the last have x of 0
        const uint32_t of_group = (uint32_t)(m * a.groups + group) * 16u + 2u * g;
        float scale0, scale1;
        if constexpr (sizeof(ST) == 2) {
          const float2 v = __half22float2(*(const __half2*)(scales + of_group * 2u));
          scale0 = v.x, scale1 = v.y;
        } else {
          const float2 v = *(const float2*)(scales + of_group * 4u);
          scale0 = v.x, scale1 = v.y;
        }
        uint32_t z0 = kOffset<H> + 0x00080008u, z1 = z0;
        if constexpr (ZP) {
          const uint32_t both = *(const uint16_t*)(zeros + of_group);
          z0 = kOffset<H> + (both & 15u) * 0x10001u, z1 = kOffset<H> + (both >> 8) * 0x10001u;
        }
        float part[NT][4] = {};
#pragma unroll
        for (int j = s * STEPS; j < (s + 1) * STEPS; ++j) {
          // words: steps 0 and 1, 2 and 3 of row g, the same of row g + 8
          const uint32_t w0 = (j < 2 ? w[m].x : w[m].y) >> (j & 1) * 8, w1 = (j < 2 ? w[m].z : w[m].w) >> (j & 1) * 8;
          uint32_t f[4];
          f[0] = minus<H>(nibbles(w0, offset), z0);
          f[1] = minus<H>(nibbles(w1, offset), z1);
          f[2] = minus<H>(nibbles(w0 >> 4, offset), z0);
          f[3] = minus<H>(nibbles(w1 >> 4, offset), z1);
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int p = SPLIT - 1; p >= 0; --p) mma<H>(part[t], f, x[t][p][2 * j], x[t][p][2 * j + 1]);
        }
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          acc[m][t][0] += part[t][0] * scale0, acc[m][t][1] += part[t][1] * scale0;
          acc[m][t][2] += part[t][2] * scale1, acc[m][t][3] += part[t][3] * scale1;
        }
      }
    }
  }

  // the warps' sums: the upper half's onto the lower half's, then those together
  auto at = [&](int m, int t, int e) -> float& { return meet[warp % (kWarps / 2)][m * 16 + g + (e >> 1) * 8][t * 8 + q * 2 + (e & 1)]; };
  if (warp >= kWarps / 2)
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) at(m, t, e) = acc[m][t][e];
  __syncthreads();
  if (warp < kWarps / 2)
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) at(m, t, e) += acc[m][t][e];
  __syncthreads();
  auto give = [&](int o, int row, float sum) {
    const int n = tile0 * 16 + o;
    if (n < a.n) ((T*)a.y)[(row0 + row) * a.n + n] = from_f32<T>(a.bias ? sum + a.bias[n] : sum);
  };
  for (int i = threadIdx.x; i < MT * 16 * rows; i += kWarps * 32) {
    const int o = i % (MT * 16), row = i / (MT * 16);
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps / 2; ++w) sum += meet[w][o][row];
    if (splits == 1) give(o, row, sum);
    else sums[i] = sum;
  }
  if (splits > 1) {  // the cluster's sums, in the order of the inputs
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    for (int i = threadIdx.x * splits + (int)cluster.block_rank(); i < MT * 16 * rows; i += kWarps * 32 * splits) {
      float sum = 0.f;
      for (int c = 0; c < splits; ++c) sum += cluster.map_shared_rank(sums, c)[i];
      give(i % (MT * 16), i / (MT * 16), sum);
    }
    cluster.sync();
  }
}

// ---- few rows of many inputs ----
// One block an SM takes an equal run of output tiles, two at a time, and its warps the inputs, the same ones of every tile: x is
// laid out once in shared memory as the lanes take it, and each warp streams its part of the codes, scales and zero points
// through a ring of its own (cp.async, a stage for up to four 64-input blocks of two tiles), so that the decoding of some hides
// behind the stream of others.
constexpr int kStreamWarps = 16;

template <int SUB, bool ZP, typename ST>
struct Stream {
  // a stage: [tile of two][block][512 bytes of codes], then [tile][block][group of the block][16 scales], then zero points alike
  static constexpr int kChunk = SUB == 4 ? 2 : 4;
  static constexpr int kScaleBytes = 16 * (int)sizeof(ST), kUnits = 2 * kChunk;
  static constexpr int kScales = kUnits * 512, kZeros = kScales + kUnits * SUB * kScaleBytes;
  static constexpr int kStage = kZeros + (ZP ? kUnits * SUB * 16 : 0);
  static constexpr int kStages = kStage * kStreamWarps * 3 <= 176 << 10 ? 3 : 2;
  static constexpr int kRing = kStage * kStages;
  static constexpr int kSums = 16 * kStreamWarps * 16 * 4;  // bytes of one of two halves: the sums of 16 tiles of a row, or of two of 8 rows
  static constexpr int kMostX = (227 << 10) - 2 * kSums - kRing * kStreamWarps;
};

__device__ __forceinline__ void stream16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

template <typename T, int SUB, bool ZP, typename ST>
__global__ void __launch_bounds__(kStreamWarps * 32, 1) linear4_stream(Linear4 a, int shift, int x_bytes) {
  using S = Stream<SUB, ZP, ST>;
  constexpr int STEPS = 4 / SUB, kChunk = S::kChunk;
  const uint32_t offset = in_register(kOffset<T>);
  extern __shared__ __align__(128) uint8_t smem[];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  const int blocks = (a.k + 63) / 64, tiles = (a.n + 15) / 16, rows = (int)a.rows;
  const int t0 = (int)((int64_t)tiles * blockIdx.x / gridDim.x), t1 = (int)((int64_t)tiles * (blockIdx.x + 1) / gridDim.x);
  const int first = (int)((int64_t)blocks * warp / kStreamWarps), last = (int)((int64_t)blocks * (warp + 1) / kStreamWarps);
  const uint32_t ring_offset = x_bytes + 2 * S::kSums + warp * S::kRing, ring_at = (uint32_t)__cvta_generic_to_shared(smem) + ring_offset;

  // the next stage to bring: tile, first block, place
  int f_tile = first < last ? t0 : t1, f_block = first;
  uint32_t f_stage = 0;
  const int tile_codes = blocks * 512;  // K below 2^24
  auto fetch = [&]() {
    if (f_tile < t1) {
      const int n = min(kChunk, last - f_block), pair = min(2, t1 - f_tile);
      const uint32_t dst = ring_at + f_stage;
      const uint8_t* const src = (const uint8_t*)a.codes + ((int64_t)f_tile * tile_codes + (f_block * 512 + lane * 16));
      if (n == kChunk && pair == 2) {
#pragma unroll
        for (int c = 0; c < kChunk; ++c) stream16(dst + lane * 16 + c * 512, src + c * 512), stream16(dst + lane * 16 + (kChunk + c) * 512, src + tile_codes + c * 512);
      } else {
        for (int m = 0; m < pair; ++m)
          for (int c = 0; c < n; ++c) stream16(dst + lane * 16 + (m * kChunk + c) * 512, src + (m * tile_codes + c * 512));
      }
      // 16 bytes a lane: groups of a block, each in sizeof(ST) pieces of scales and one of zero points
      auto group_of = [&](int c, int s) { return SUB == 1 ? (f_block + c) >> shift : min((f_block + c) * SUB + s, a.groups - 1); };  // behind the last x is 0
#pragma unroll
      for (int i0 = 0; i0 < S::kUnits * SUB * (int)sizeof(ST); i0 += 32) {
        const int i = i0 + lane, piece = i % (int)sizeof(ST), s = i / (int)sizeof(ST) % SUB, c = i / ((int)sizeof(ST) * SUB) % kChunk, m = i / ((int)sizeof(ST) * SUB * kChunk);
        if (m < pair && c < n) stream16(dst + S::kScales + i * 16, (const uint8_t*)a.scales + (((int64_t)(f_tile + m) * a.groups + group_of(c, s)) * S::kScaleBytes + piece * 16));
      }
      if constexpr (ZP) {
#pragma unroll
        for (int i0 = 0; i0 < S::kUnits * SUB; i0 += 32) {
          const int i = i0 + lane, s = i % SUB, c = i / SUB % kChunk, m = i / (SUB * kChunk);
          if (m < pair && c < n) stream16(dst + S::kZeros + i * 16, a.zeros + ((int64_t)(f_tile + m) * a.groups + group_of(c, s)) * 16);
        }
      }
      f_stage = f_stage + S::kStage == (uint32_t)S::kRing ? 0 : f_stage + S::kStage;
      f_block += n;
      if (f_block == last) f_block = first, f_tile += 2;
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  // the weights are the session's own: they need not wait for the kernel in front
#pragma unroll
  for (int i = 0; i < S::kStages; ++i) fetch();
  asm volatile("griddepcontrol.wait;" ::: "memory");

  // x as [steps 0 and 1, 2 and 3][row][block][lane of a quarter][8], zeros behind K; an odd number of blocks keeps rows on other banks
  const int row_bytes = (blocks | 1) * 64, half_bytes = rows * row_bytes;
  const bool whole = a.k % 8 == 0 && ((uintptr_t)a.x & 15) == 0;
  constexpr int kAtOnce = 4;  // rows whose loads are in flight together
#pragma unroll 1
  for (int i = threadIdx.x; i < blocks * 8; i += kStreamWarps * 32) {  // 8 lanes of x: two lanes of a quarter
    uint8_t* const dst = smem + (i >> 2 & 1) * half_bytes + (i >> 3) * 64 + (i & 1) * 32 + (i >> 1 & 1) * 8;
#pragma unroll 1
    for (int row0 = 0; row0 < rows; row0 += kAtOnce) {
      const T* const src = (const T*)a.x + ((int64_t)row0 * a.k + i * 8);
      uint4 v[kAtOnce];
#pragma unroll
      for (int r = 0; r < kAtOnce; ++r) {
        v[r] = make_uint4(0, 0, 0, 0);
        if (row0 + r >= rows) continue;
        if (whole) {
          if (i * 8 < a.k) v[r] = *(const uint4*)(src + (int64_t)r * a.k);
        } else {
          uint32_t w[1][8];
          load4<T, 1>(src + (int64_t)r * a.k, a.k - i * 8, false, w, 0);
          load4<T, 1>(src + (int64_t)r * a.k + 4, a.k - i * 8 - 4, false, w, 2);
          v[r] = make_uint4(w[0][0], w[0][1], w[0][2], w[0][3]);
        }
      }
#pragma unroll
      for (int r = 0; r < kAtOnce; ++r)
        if (row0 + r < rows) {
          *(uint2*)(dst + (row0 + r) * row_bytes) = make_uint2(v[r].x, v[r].y);
          *(uint2*)(dst + (row0 + r) * row_bytes + 16) = make_uint2(v[r].z, v[r].w);
        }
    }
  }
  __syncthreads();
  const uint32_t x_at = min(g, rows - 1) * row_bytes + q * 16;  // rows behind the last are copies of it: their columns of the products go nowhere

  uint32_t stage = 0;
  int slot = 0, half = 0;
  const int slots = 16 / rows & ~1;  // tiles whose sums meet at a time: two at least
  for (int tile = t0; tile < t1; tile += 2) {
    const bool two = tile + 1 < t1;
    float acc[2][4] = {};
    for (int b0 = first; b0 < last; b0 += kChunk) {
      asm volatile("cp.async.wait_group %0;" ::"n"(S::kStages - 1) : "memory");
      __syncwarp();
      const uint8_t *const at = smem + ring_offset + stage, *const codes = at + lane * 16, *const scales = at + S::kScales + 2 * g * (int)sizeof(ST), *const zeros = at + S::kZeros + 2 * g;
      stage = stage + S::kStage == (uint32_t)S::kRing ? 0 : stage + S::kStage;
      auto x_of = [&](int c, uint32_t (&x)[8]) {
        const uint8_t* const src = smem + (x_at + b0 * 64) + c * 64;
        *(uint4*)&x[0] = *(const uint4*)src;
        *(uint4*)&x[4] = *(const uint4*)(src + half_bytes);
      };
      auto unit = [&](int m, int c, const uint32_t (&x)[8], float (&sum)[4]) {
        const int u = m * kChunk + c;
        const uint4 w = *(const uint4*)(codes + u * 512);
#pragma unroll
        for (int s = 0; s < SUB; ++s) {
          float scale0, scale1;
          if constexpr (sizeof(ST) == 2) {
            const float2 v = __half22float2(*(const __half2*)(scales + (u * SUB + s) * S::kScaleBytes));
            scale0 = v.x, scale1 = v.y;
          } else {
            const float2 v = *(const float2*)(scales + (u * SUB + s) * S::kScaleBytes);
            scale0 = v.x, scale1 = v.y;
          }
          uint32_t z0 = kOffset<T> + 0x00080008u, z1 = z0;
          if constexpr (ZP) {
            const uint32_t both = *(const uint16_t*)(zeros + (u * SUB + s) * 16);
            z0 = kOffset<T> + (both & 15u) * 0x10001u, z1 = kOffset<T> + (both >> 8) * 0x10001u;
          }
          float part[4] = {};
#pragma unroll
          for (int j = s * STEPS; j < (s + 1) * STEPS; ++j) {
            const uint32_t w0 = (j < 2 ? w.x : w.y) >> (j & 1) * 8, w1 = (j < 2 ? w.z : w.w) >> (j & 1) * 8;
            uint32_t f[4];
            f[0] = minus<T>(nibbles(w0, offset), z0);
            f[1] = minus<T>(nibbles(w1, offset), z1);
            f[2] = minus<T>(nibbles(w0 >> 4, offset), z0);
            f[3] = minus<T>(nibbles(w1 >> 4, offset), z1);
            mma<T>(part, f, x[2 * j], x[2 * j + 1]);
          }
          sum[0] += part[0] * scale0, sum[1] += part[1] * scale0;
          sum[2] += part[2] * scale1, sum[3] += part[3] * scale1;
        }
      };
      auto units = [&](auto count) {  // without a branch between them, so that they overlap
#pragma unroll
        for (int c = 0; c < decltype(count)::value; ++c) {
          uint32_t x[8];
          x_of(c, x);
          unit(0, c, x, acc[0]);
          unit(1, c, x, acc[1]);
        }
      };
      const int n = min(kChunk, last - b0);
      if (two && n == kChunk) {
        units(std::integral_constant<int, kChunk>());
      } else if (two && n == 3 && kChunk > 3) {
        units(std::integral_constant<int, 3>());
      } else if (two && n == 2) {
        units(std::integral_constant<int, 2>());
      } else {
#pragma unroll 1
        for (int c = 0; c < n; ++c) {
          uint32_t x[8];
          x_of(c, x);
          unit(0, c, x, acc[0]);
          if (two) unit(1, c, x, acc[1]);
        }
      }
      __syncwarp();  // all lanes have read the stage
      fetch();
    }
    float* const meet = (float*)(smem + x_bytes + half * S::kSums);
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int row = q * 2 + (e & 1);
        if (row < rows) meet[(((slot + m) * kStreamWarps + warp) * rows + row) * 16 + g + (e >> 1) * 8] = acc[m][e];
      }
    slot += 2;
    if (slot < slots && tile + 2 < t1) continue;
    __syncthreads();  // the other half's sums have been taken: who takes them passes here afterwards
    for (int i = threadIdx.x; i < slot * rows * 16; i += kStreamWarps * 32) {
      const int o = i % 16, row = i / 16 % rows, which = i / 16 / rows, n = (tile + 2 - slot + which) * 16 + o;
      float sum = 0.f;
#pragma unroll
      for (int w = 0; w < kStreamWarps; ++w) sum += meet[((which * kStreamWarps + w) * rows + row) * 16 + o];
      if (n < min(a.n, t1 * 16)) ((T*)a.y)[(int64_t)row * a.n + n] = from_f32<T>(a.bias ? sum + a.bias[n] : sum);
    }
    slot = 0, half ^= 1;
  }
}

template <typename T, int SUB, bool ZP, typename ST>
bool launch_stream(const Linear4& a, cudaStream_t s) {
  using S = Stream<SUB, ZP, ST>;
  const int64_t x_bytes = a.rows * (ceil_div(a.k, 64) | 1) * 128;
  if (x_bytes > S::kMostX) return false;
  static std::mutex mu;
  static bool have[64] = {};
  int device = 0, shift = 0;
  OXB_CUDA(cudaGetDevice(&device));
  {
    std::lock_guard<std::mutex> lock(mu);
    if (device < 0 || device >= 64 || !have[device]) {
      OXB_CUDA(cudaFuncSetAttribute(linear4_stream<T, SUB, ZP, ST>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kMostX + 2 * S::kSums + S::kRing * kStreamWarps));
      if (device >= 0 && device < 64) have[device] = true;
    }
  }
  while ((64 << shift) < a.group) ++shift;
  launch(linear4_stream<T, SUB, ZP, ST>, dim3((unsigned)std::min<int64_t>(device_sms(), ceil_div(a.n, 16))), dim3(kStreamWarps * 32),
         (size_t)x_bytes + 2 * S::kSums + S::kRing * kStreamWarps, s, a, shift, (int)x_bytes);
  return true;
}
template <typename T, int SUB>
bool launch_stream(const Linear4& a, cudaStream_t s) {
  if (a.scales_f16) return a.zeros ? launch_stream<T, SUB, true, __half>(a, s) : launch_stream<T, SUB, false, __half>(a, s);
  return a.zeros ? launch_stream<T, SUB, true, float>(a, s) : launch_stream<T, SUB, false, float>(a, s);
}
template <typename T>
bool launch_stream(const Linear4& a, cudaStream_t s) {  // false: x does not fit
  return a.group == 16 ? launch_stream<T, 4>(a, s) : a.group == 32 ? launch_stream<T, 2>(a, s) : launch_stream<T, 1>(a, s);
}

template <typename T, int MT, int NT, int SUB, bool ZP, typename ST>
void launch_rows(const Linear4& a, int64_t row0, int64_t rows, cudaStream_t s) {
  // The inputs are split over as many blocks as bring the grid to two blocks an SM, while a warp keeps two 64-input blocks.
  const int64_t outputs = ceil_div(ceil_div(a.n, 16), MT), row_blocks = ceil_div(rows, NT * 8), blocks = ceil_div(a.k, 64);
  int splits = 1, shift = 0;
  while (splits < 8 && outputs * row_blocks * splits * 2 <= 2 * device_sms() && blocks >= 2LL * kWarps * splits * 2) splits *= 2;
  while ((64 << shift) < a.group) ++shift;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(outputs * splits), (unsigned)row_blocks);
  cfg.blockDim = dim3(kWarps * 32);
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = splits;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = splits > 1 ? 2 : 1;
  OXB_CUDA(cudaLaunchKernelEx(&cfg, linear4_rows<T, MT, NT, SUB, ZP, ST>, a, row0, shift, splits));
}
template <typename T, int MT, int NT, int SUB>
void launch_rows(const Linear4& a, int64_t row0, int64_t rows, cudaStream_t s) {
  if (a.scales_f16) a.zeros ? launch_rows<T, MT, NT, SUB, true, __half>(a, row0, rows, s) : launch_rows<T, MT, NT, SUB, false, __half>(a, row0, rows, s);
  else a.zeros ? launch_rows<T, MT, NT, SUB, true, float>(a, row0, rows, s) : launch_rows<T, MT, NT, SUB, false, float>(a, row0, rows, s);
}
template <typename T, int MT, int NT>
void launch_rows(const Linear4& a, int64_t row0, int64_t rows, cudaStream_t s) {
  if (a.group == 16) launch_rows<T, MT, NT, 4>(a, row0, rows, s);
  else if (a.group == 32) launch_rows<T, MT, NT, 2>(a, row0, rows, s);
  else launch_rows<T, MT, NT, 1>(a, row0, rows, s);
}
template <typename T>
void launch_rows(const Linear4& a, cudaStream_t s) {
  // Tiles of 16 outputs for a warp, in us at rows x K x N, 1 / 2 / 4 tiles: 1 x 1024 x 16384 5.8 / 5.3 / 3.8, 4 x 4096 x 16384
  // (f32) 32 / 25 / 18, 8 x 2048 x 8192 7.6 / 5.4 / 5.5, where rows are fetched once for all of them; with two fragments of rows
  // 16 x 4096 x 4096 10.3 / 7.2 / 8.2, 32 x 4096 x 4096 (f32) 32 / 22 / 25, but 16 x 4096 x 16384 - / 17.2 / 14.0, whose outputs alone
  // give every SM a block of 4; small matrices want the blocks: 1 x 1024 x 1024
  // 2.3 / 2.5 / 3.0, 5 x 1000 x 1111 (f32) 3.6 / 3.9 / 4.5.
  const bool large = (int64_t)a.n * a.k >= 148LL * 65536;
  // The stream against the blocks below, in us: 1 x 4096 x 16384 10.0 / 11.5, 4 rows 10.8 / 11.8, 1 x 4096 x 4096 4.0 / 4.9,
  // 1 x 4096 x 65536 30 / 44, 1 x 2048 x 2048 2.8 / 4.2, 8 rows 3.4 / 5.2, 1 x 2880 x 5120 5.1 / 5.8; with few inputs a warp's turn
  // is too short: 1 x 2048 x 16384 7.8 / 6.4, 1 x 1024 x 1024 2.2 / 2.3, 1 x 512 x 2048 2.5 / 2.0.
  if constexpr (sizeof(T) == 2)
    if (a.rows <= 8 && a.k >= (large ? 2560 : 2048) && launch_stream<T>(a, s)) return;
  // grid.y holds 65535 blocks of rows
  for (int64_t row0 = 0; row0 < a.rows; row0 += 65535LL * 16) {
    const int64_t rows = std::min<int64_t>(a.rows - row0, 65535LL * 16);
    if (rows <= 8) large ? launch_rows<T, 4, 1>(a, row0, rows, s) : launch_rows<T, 1, 1>(a, row0, rows, s);
    else if (rows <= 16 || sizeof(T) == 4) large ? a.n >= 64 * 148 ? launch_rows<T, 4, 2>(a, row0, rows, s) : launch_rows<T, 2, 2>(a, row0, rows, s) : launch_rows<T, 1, 2>(a, row0, rows, s);
    else if constexpr (sizeof(T) == 2) launch_rows<T, 1, 4>(a, row0, rows, s);  // of exact weights

  }
}

}  // namespace

// 16-bit rows from here on run on tcgen05 (umma_linear4.cu), whose block takes 128 outputs by up to 256 rows.  This file's kernel
// against that one, at 4096x4096: 16 rows 7.2 / 9.8 us, 32 rows 13.0 / 10.2, 64 rows 24.9 / 10.4.
constexpr int64_t kManyRows = 17;

bool linear4_many_rows(const Linear4& a) { return a.dt != DT::F32 && a.rows >= kManyRows && !a.exact_weights; }

void linear4(const Linear4& a, cudaStream_t s) {
  if (a.rows == 0) return;
  if (linear4_many_rows(a)) linear4_prompt(a, s);
  else if (a.dt == DT::F32) launch_rows<float>(a, s);
  else if (a.dt == DT::F16) launch_rows<__half>(a, s);
  else launch_rows<__nv_bfloat16>(a, s);
}

}  // namespace k
}  // namespace oxb
