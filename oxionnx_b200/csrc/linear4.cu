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
// A block has 16 (or 64) outputs and splits the inputs over its warps; the warps' sums meet in shared memory in one order.
// 1 x 4096 x 16384 takes 12.5 us, where the codes alone stream in 7.3: the decoding (about 106 instructions for 16 outputs by 64
// inputs) is not hidden entirely.
#include <cooperative_groups.h>

#include <algorithm>

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

// A nibble in the low bits of a number whose last place is 1: 128 + code in bf16, 1024 + code in f16.
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
          f[0] = minus<H>((w0 & 0x000f000fu) | kOffset<H>, z0);
          f[1] = minus<H>((w1 & 0x000f000fu) | kOffset<H>, z1);
          f[2] = minus<H>((w0 >> 4 & 0x000f000fu) | kOffset<H>, z0);
          f[3] = minus<H>((w1 >> 4 & 0x000f000fu) | kOffset<H>, z1);
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
  // Tiles of 16 outputs for a warp, in us at rows x K x N, 1 / 2 / 4 tiles: 1 x 4096 x 16384 17.9 / 13.4 / 12.5, 8 x 4096 x 4096
  // 10.9 / 8.9 / 6.4, 16 x 4096 x 4096 10.8 / 10.1 / 8.5, where rows are fetched once for all of them; small matrices want the
  // blocks: 1 x 1024 x 1024 2.3 / 2.5 / 3.0, 5 x 1000 x 1111 (f32) 3.6 / 3.9 / 4.5; and so do 32 rows, whose fragments fill the
  // registers: 32 x 4096 x 4096 12.9 / 16.2 / 18.2.
  const bool large = (int64_t)a.n * a.k >= 148LL * 65536;
  // grid.y holds 65535 blocks of rows
  for (int64_t row0 = 0; row0 < a.rows; row0 += 65535LL * 16) {
    const int64_t rows = std::min<int64_t>(a.rows - row0, 65535LL * 16);
    if (rows <= 8) large ? launch_rows<T, 4, 1>(a, row0, rows, s) : launch_rows<T, 1, 1>(a, row0, rows, s);
    else if (rows <= 16 || sizeof(T) == 4) large ? launch_rows<T, 4, 2>(a, row0, rows, s) : launch_rows<T, 1, 2>(a, row0, rows, s);
    else launch_rows<T, 1, 4>(a, row0, rows, s);
  }
}

}  // namespace

// 16-bit rows from here on run on tcgen05 (umma_linear4.cu), whose block takes 128 outputs by up to 256 rows.  This file's kernel
// against that one, at 4096x4096: 16 rows 8.5 / 9.8 us, 32 rows 13.0 / 10.2, 64 rows 24.9 / 10.4.
constexpr int64_t kManyRows = 17;

bool linear4_many_rows(const Linear4& a) { return a.dt != DT::F32 && a.rows >= kManyRows; }

void linear4(const Linear4& a, cudaStream_t s) {
  if (a.rows == 0) return;
  if (linear4_many_rows(a)) linear4_prompt(a, s);
  else if (a.dt == DT::F32) launch_rows<float>(a, s);
  else if (a.dt == DT::F16) launch_rows<__half>(a, s);
  else launch_rows<__nv_bfloat16>(a, s);
}

}  // namespace k
}  // namespace oxb
