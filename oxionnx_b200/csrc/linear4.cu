// Rows times a matrix of 4-bit codes with a scale (and a zero point) for each group of inputs,
//   y[m][n] = sum over groups g of scale[n][g] * sum over k in g of x[m][k] (code[n][k] - zero[n][g])  + bias[n],
// for few rows: what bounds it is reading the codes once.
//
// The codes are laid out once, when a session is planned, in the order in which the lanes of a warp take them (Linear4Layout):
// 16 bytes a lane are the m16n8k16 fragments of 16 outputs by 64 inputs.  Outputs are the fragments' rows and x's rows their
// columns, so that up to 8 rows cost no more instructions than one.  code - zero is a whole number below 16 in size and exact
// in either 16-bit type, so the products are exact and the sums are f32; a group's sum is scaled in f32.  f32 rows are taken
// as the sum of three bf16 numbers (8 bits of the significand each, all 24 of them), whose products are exact as well.
//
// A block has 16 (or 32) outputs and splits the inputs over its warps; the warps' sums meet in shared memory in one order.
#include <algorithm>

#include "decoder_device.cuh"

namespace oxb {
namespace k {

namespace {

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
__device__ __forceinline__ void load4(const T* src, int left, uint32_t (&w)[SPLIT][8], int at, bool aligned) {
  if constexpr (sizeof(T) == 2) {
    if (left >= 4 && aligned) {
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
    if (left >= 4 && aligned) {
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
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        w[s][at + i] = *(const uint32_t*)&h;
        // an infinity's remainder is 0, not infinity minus infinity; NaN stays in the first part
        const float ra = a - __low2float(h), rb = b - __high2float(h);
        a = fabsf(a) <= 3.4028235e38f && fabsf(ra) <= 3.4028235e38f ? ra : 0.f;
        b = fabsf(b) <= 3.4028235e38f && fabsf(rb) <= 3.4028235e38f ? rb : 0.f;
      }
    }
  }
}

// MT: tiles of 16 outputs; NT: of 8 rows; SUB: groups of a 64-input block (4, 2 or 1); ST: type of the scales.
template <typename T, int MT, int NT, int SUB, typename ST>
__global__ void __launch_bounds__(kWarps * 32) linear4_rows(Linear4 a, int64_t row0) {
  using H = typename Operand<T>::type;
  constexpr int SPLIT = sizeof(T) == 4 ? 3 : 1, STEPS = 4 / SUB;  // k16 steps of a group within the block
  extern __shared__ float meet[];                                 // [warp][MT * 16 outputs][NT * 8 rows + 1]
  pdl_enter();
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  const int tile0 = blockIdx.x * MT, tiles = (a.n + 15) / 16, blocks = (a.k + 63) / 64;
  row0 += (int64_t)blockIdx.y * NT * 8;
  const int first = (int)((int64_t)blocks * warp / kWarps), last = (int)((int64_t)blocks * (warp + 1) / kWarps);
  const int rows = (int)min((int64_t)NT * 8, a.rows - row0);
  const bool aligned = a.k % 4 == 0 && ((uintptr_t)a.x & 15) == 0;

  float acc[MT][NT][4] = {};
  const uint4* codes[MT];
  const ST* scales[MT];
  const uint8_t* zeros[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const int64_t tile = min(tile0 + m, tiles - 1);
    codes[m] = (const uint4*)a.codes + tile * blocks * 32 + lane;
    scales[m] = (const ST*)a.scales + tile * a.groups * 16 + 2 * g;
    zeros[m] = a.zeros ? a.zeros + tile * a.groups * 16 + 2 * g : nullptr;
  }
#pragma unroll 2
  for (int b = first; b < last; ++b) {
    uint4 w[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) w[m] = __ldcs(codes[m] + (int64_t)b * 32);
    uint32_t x[NT][SPLIT][8];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int row = t * 8 + g;
      const bool real = row < rows;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int k = b * 64 + j * 16 + q * 4;
        load4<T, SPLIT>((const T*)a.x + (real && k < a.k ? (row0 + row) * a.k + k : 0), real ? a.k - k : 0, x[t], 2 * j, aligned);
      }
    }
#pragma unroll
    for (int m = 0; m < MT; ++m) {
#pragma unroll
      for (int s = 0; s < SUB; ++s) {
        const int group = SUB == 1 ? b * 64 / a.group : min(b * SUB + s, a.groups - 1);  // of a block's groups behind the last, the codes are zeros' and x is 0
        const ST* const sc = scales[m] + (int64_t)group * 16;
        const float scale0 = to_f32(sc[0]), scale1 = to_f32(sc[1]);
        uint32_t z0 = kOffset<H> + 0x00080008u, z1 = z0;
        if (zeros[m]) {
          const uint32_t both = *(const uint16_t*)(zeros[m] + (int64_t)group * 16);
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
  constexpr int LD = NT * 8 + 1;
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) meet[(warp * MT * 16 + m * 16 + g + (e >> 1) * 8) * LD + t * 8 + q * 2 + (e & 1)] = acc[m][t][e];
  __syncthreads();
  for (int i = threadIdx.x; i < MT * 16 * rows; i += kWarps * 32) {
    const int o = i % (MT * 16), row = i / (MT * 16), n = tile0 * 16 + o;
    if (n >= a.n) continue;
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) sum += meet[(w * MT * 16 + o) * LD + row];
    ((T*)a.y)[(row0 + row) * a.n + n] = from_f32<T>(a.bias ? sum + a.bias[n] : sum);
  }
}

template <typename T, int MT, int NT, int SUB, typename ST>
void launch_rows(const Linear4& a, int64_t row0, int64_t rows, cudaStream_t s) {
  const size_t smem = (size_t)kWarps * MT * 16 * (NT * 8 + 1) * sizeof(float);
  static_assert((size_t)kWarps * MT * 16 * (NT * 8 + 1) * sizeof(float) <= 48 * 1024, "no opt-in");
  const dim3 grid((unsigned)ceil_div(ceil_div(a.n, 16), MT), (unsigned)ceil_div(rows, NT * 8));
  launch(linear4_rows<T, MT, NT, SUB, ST>, grid, dim3(kWarps * 32), smem, s, a, row0);
}
template <typename T, int MT, int NT, int SUB>
void launch_rows(const Linear4& a, int64_t row0, int64_t rows, cudaStream_t s) {
  a.scales_f16 ? launch_rows<T, MT, NT, SUB, __half>(a, row0, rows, s) : launch_rows<T, MT, NT, SUB, float>(a, row0, rows, s);
}
template <typename T, int MT, int NT>
void launch_rows(const Linear4& a, int64_t row0, int64_t rows, cudaStream_t s) {
  if (a.group == 16) launch_rows<T, MT, NT, 4>(a, row0, rows, s);
  else if (a.group == 32) launch_rows<T, MT, NT, 2>(a, row0, rows, s);
  else launch_rows<T, MT, NT, 1>(a, row0, rows, s);
}
template <typename T>
void launch_rows(const Linear4& a, cudaStream_t s) {
  // grid.y holds 65535 blocks of rows
  for (int64_t row0 = 0; row0 < a.rows; row0 += 65535LL * 16) {
    const int64_t rows = std::min<int64_t>(a.rows - row0, 65535LL * 16);
    if (rows <= 8) launch_rows<T, 1, 1>(a, row0, rows, s);
    else if (rows <= 16 || sizeof(T) == 4) launch_rows<T, 2, 2>(a, row0, rows, s);
    else launch_rows<T, 2, 4>(a, row0, rows, s);
  }
}

}  // namespace

void linear4(const Linear4& a, cudaStream_t s) {
  if (a.rows == 0) return;
  if (a.dt == DT::F32) launch_rows<float>(a, s);
  else if (a.dt == DT::F16) launch_rows<__half>(a, s);
  else launch_rows<__nv_bfloat16>(a, s);
}

}  // namespace k
}  // namespace oxb
