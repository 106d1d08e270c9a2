// Many 16-bit rows times a matrix of 4-bit codes, on tcgen05: the matrix stays in 4 bits in memory and becomes 16-bit lanes on
// its way into the products.
//
// A block has 128 outputs and up to 256 rows of x.  Outputs are the rows of the accumulator, so that a weight is an element of
// the A operand, which tensor memory may hold: the thread of an output decodes 64 of its codes, (code - zero) * scale rounded
// once to x's type, and writes them there, a store of 32 columns and no shared memory.  x comes through TMA as the B operand.
// Sixteen warps decode (four a block of 64 inputs, in turns), one thread brings x, one issues the products, which for a block
// of 64 inputs by 256 rows take 512 cycles.  With eight warps a block of inputs took 800, as long as one's decoding; with
// sixteen 650: 2048 x 4096 x 4096 takes 62 us, 1110 TFLOP/s, in two turns of 256 tiles over 148 SMs.
//
// The roundings of the weights are as large as those of the result (half a step of x's type each, and independent).  For that
// they have to be normal numbers of x's type: outputs with scales that would leave it bring a power of two with them, which
// the sums are multiplied by in the end (linear4_folds).
// Every wait is bounded.
#include <cooperative_groups.h>

#include <algorithm>
#include <cmath>
#include <mutex>
#include <type_traits>
#include <vector>

#include "decoder_device.cuh"
#include "umma_kernel.cuh"

namespace oxb {
namespace k {

namespace umma {

namespace cg = cooperative_groups;

constexpr int L4_OUTPUTS = 128, L4_K = 64;
constexpr int L4_GROUPS = 4;  // of four warps that decode
constexpr int L4_THREADS = L4_GROUPS * 128 + 64;
constexpr int L4_WEIGHT_STAGES = 8;  // 32 columns of tensor memory each

template <int ROWS>
struct Linear4Shape {
  static constexpr uint32_t kTile = ROWS * 128u;  // rows of 64 lanes
  static constexpr int kStages = ROWS == 256 ? 6 : 8;
  static constexpr uint32_t kSmem = kStages * kTile + 1024u;
  static constexpr uint32_t kAcc = 0, kWeights = 256;  // columns of tensor memory
  static_assert(kStages * kTile >= ROWS * 512u, "the sums of a cluster meet where x was");
};

struct alignas(64) Linear4Params {
  CUtensorMap x;
  Linear4 a;
  int blocks, shift;  // of 64 inputs; log2 of the inputs of a group
  int splits;         // blocks of a cluster, which share an output tile's inputs
  uint32_t idesc;
};

// Weights out of codes: (code - zero) * scale, rounded once.  code - zero is exact in both types.
template <typename T, typename ST>
struct Decoder;  // f32 scales: products in f32
template <>
struct Decoder<__half, float> {
  uint32_t zero;
  float scale;
  __device__ __forceinline__ Decoder(uint32_t z, float s) : zero(0x64006400u + z * 0x10001u), scale(s) {}
  __device__ __forceinline__ uint32_t operator()(uint32_t w, uint32_t offset) const {
    const uint32_t v = nibbles(w, offset);
    const float2 d = __half22float2(__hsub2(*(const __half2*)&v, *(const __half2*)&zero));
    const __half2 r = __floats2half2_rn(d.x * scale, d.y * scale);
    return *(const uint32_t*)&r;
  }
};
template <>
struct Decoder<__nv_bfloat16, float> {
  uint32_t zero;
  float scale;
  __device__ __forceinline__ Decoder(uint32_t z, float s) : zero(0x43004300u + z * 0x10001u), scale(s) {}
  __device__ __forceinline__ uint32_t operator()(uint32_t w, uint32_t offset) const {
    const uint32_t v = nibbles(w, offset);
    const __nv_bfloat162 d = __hsub2(*(const __nv_bfloat162*)&v, *(const __nv_bfloat162*)&zero);
    const uint32_t x = *(const uint32_t*)&d;
    const __nv_bfloat162 r = __floats2bfloat162_rn(__uint_as_float(x << 16) * scale, __uint_as_float(x & 0xffff0000u) * scale);
    return *(const uint32_t*)&r;
  }
};
// f16 scales: one f16 product
template <>
struct Decoder<__half, __half> {
  uint32_t zero;
  __half2 scale;
  __device__ __forceinline__ Decoder(uint32_t z, __half s) : zero(0x64006400u + z * 0x10001u), scale(__half2half2(s)) {}
  __device__ __forceinline__ uint32_t operator()(uint32_t w, uint32_t offset) const {
    const uint32_t v = nibbles(w, offset);
    const __half2 r = __hmul2(__hsub2(*(const __half2*)&v, *(const __half2*)&zero), scale);
    return *(const uint32_t*)&r;
  }
};
// An f16 scale is the sum of two bf16 numbers, of 8 bits and of what is left, at most 3.  The second's product with a number
// below 16 has 7 bits and is exact, so that adding it to the first's is the only rounding.
template <>
struct Decoder<__nv_bfloat16, __half> {
  uint32_t zero;
  __nv_bfloat162 high, low;
  __device__ __forceinline__ Decoder(uint32_t z, __half s) : zero(0x43004300u + z * 0x10001u) {
    const float f = __half2float(s);
    const __nv_bfloat16 h = __float2bfloat16_rn(f);
    high = __bfloat162bfloat162(h);
    low = __bfloat162bfloat162(__float2bfloat16_rn(f - __bfloat162float(h)));
  }
  __device__ __forceinline__ uint32_t operator()(uint32_t w, uint32_t offset) const {
    const uint32_t v = nibbles(w, offset);
    const __nv_bfloat162 d = __hsub2(*(const __nv_bfloat162*)&v, *(const __nv_bfloat162*)&zero), r = __hfma2(d, high, __hmul2(d, low));
    return *(const uint32_t*)&r;
  }
};

__device__ __forceinline__ void l4_mma(uint32_t tmem_d, uint32_t tmem_a, uint64_t db, uint32_t idesc, uint32_t accumulate) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(tmem_d), "r"(tmem_a), "l"(db), "r"(idesc),
               "r"(accumulate)
               : "memory");
}
__device__ __forceinline__ void l4_store32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
      "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}

// WIDE: a group is at least a block of 64 inputs, which then has one scale.
template <typename T, int ROWS, typename ST, bool WIDE>
__global__ void __launch_bounds__(L4_THREADS, 1) umma_linear4_kernel(const __grid_constant__ Linear4Params p) {
  using S = Linear4Shape<ROWS>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t bar_x_full[S::kStages], bar_x_empty[S::kStages], bar_w_full[L4_WEIGHT_STAGES], bar_w_empty[L4_WEIGHT_STAGES], bar_acc;
  __shared__ uint32_t tmem_base_slot;
  __shared__ int abort_flag;
  const Linear4& a = p.a;
  const int warp = (int)(threadIdx.x >> 5), lane = (int)(threadIdx.x & 31);
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* const base_ptr = smem_raw + (base - smem_u32(smem_raw));
  volatile int* const abortp = &abort_flag;
  const int out_blocks = (a.n + L4_OUTPUTS - 1) / L4_OUTPUTS;
  const int tile_of_grid = blockIdx.x / p.splits, split = blockIdx.x % p.splits;
  const int out0 = tile_of_grid % out_blocks * L4_OUTPUTS;
  const int64_t row0 = (int64_t)(tile_of_grid / out_blocks) * ROWS;
  const int block0 = (int)((int64_t)p.blocks * split / p.splits), blocks = (int)((int64_t)p.blocks * (split + 1) / p.splits) - block0;  // its inputs
  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int i = 0; i < S::kStages; ++i) mbar_init(smem_u32(&bar_x_full[i]), 1), mbar_init(smem_u32(&bar_x_empty[i]), 1);
    for (int i = 0; i < L4_WEIGHT_STAGES; ++i) mbar_init(smem_u32(&bar_w_full[i]), 4), mbar_init(smem_u32(&bar_w_empty[i]), 1);
    mbar_init(smem_u32(&bar_acc), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 4 * L4_GROUPS) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base_slot)), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_base_slot;
  pdl_enter();
  auto give_up = [&](int code) {
    if (!*abortp) {
      *abortp = 1;
      atomicExch(a.err, code);
    }
  };

  if (warp == 4 * L4_GROUPS + 1) {
    // ---------------- rows of x ----------------
    if (elect_one()) {
      for (int b = 0; b < blocks; ++b) {
        const int stage = b % S::kStages;
        if (b >= S::kStages && !mbar_wait(smem_u32(&bar_x_empty[stage]), ((b / S::kStages) & 1u) ^ 1u, abortp)) {
          give_up(61);
          break;
        }
        mbar_expect_tx(smem_u32(&bar_x_full[stage]), S::kTile);
        tma_load_2d(base + stage * S::kTile, &p.x, smem_u32(&bar_x_full[stage]), (block0 + b) * L4_K, (int)row0);
      }
    }
    __syncwarp();
  } else if (warp == 4 * L4_GROUPS) {
    // ---------------- products ----------------
    if (elect_one()) {
      const uint64_t x_at = make_smem_desc(base, 128);
      const uint32_t w_at = tmem + S::kWeights, acc = tmem + S::kAcc, idesc = p.idesc;
      bool ok = true;
      for (int b = 0; b < blocks; ++b) {
        const int stage = b % S::kStages, ws = b % L4_WEIGHT_STAGES;
        ok = mbar_wait(smem_u32(&bar_x_full[stage]), (b / S::kStages) & 1u, abortp) && mbar_wait(smem_u32(&bar_w_full[ws]), (b / L4_WEIGHT_STAGES) & 1u, abortp);
        if (!ok) {
          give_up(62);
          break;
        }
        tc_fence_after();
        const uint64_t at = x_at + (uint32_t)stage * (S::kTile >> 4);
#pragma unroll
        for (int k = 0; k < L4_K / 16; ++k) l4_mma(acc, w_at + ws * 32 + k * 8, at + 2 * k, idesc, k > 0 ? 1u : (b > 0 ? 1u : 0u));
        tc_commit<false>(smem_u32(&bar_x_empty[stage]));
        tc_commit<false>(smem_u32(&bar_w_empty[ws]));
      }
      if (ok) tc_commit<false>(smem_u32(&bar_acc));
    }
    __syncwarp();
  } else {
    // ---------------- weights, then the rows' way out ----------------
    const int turn = warp >> 2, quarter = warp & 3, r = quarter * 32 + lane;
    const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
    const int tiles = (a.n + 63) / 64 * 4, tile = min((out0 + r) / 16, tiles - 1), in_tile = r % 8 * 2 + r % 16 / 8;
    const uint8_t* const codes = (const uint8_t*)a.codes + (int64_t)tile * p.blocks * 512 + r % 8 * 64 + r % 16 / 8 * 8;
    const ST* const scales = (const ST*)a.scales + (int64_t)tile * a.groups * 16 + in_tile;
    const uint8_t* const zeros = a.zeros ? a.zeros + (int64_t)tile * a.groups * 16 + in_tile : nullptr;
    // what a block of 64 inputs takes, fetched while the one before is decoded
    constexpr int SCALES = WIDE ? 1 : 4;
    struct Fetched {
      uint2 codes[4];
      ST scale[SCALES];  // of the block, or of its four 16 inputs; those behind the last group meet x of 0
      uint8_t zero[SCALES];
    } next;
    auto fetch = [&](int local) {
      const int b = block0 + local;
#pragma unroll
      for (int q = 0; q < 4; ++q) next.codes[q] = *(const uint2*)(codes + (int64_t)b * 512 + q * 16);
#pragma unroll
      for (int s = 0; s < SCALES; ++s) {
        const int at = (WIDE ? b >> (p.shift - 6) : min((b * 64 + s * 16) >> p.shift, a.groups - 1)) * 16;
        next.scale[s] = scales[at];
        next.zero[s] = zeros ? zeros[at] : (uint8_t)8;
      }
    };
    if (turn < blocks) fetch(turn);
    const uint32_t offset = in_register(std::is_same<T, __half>::value ? 0x64006400u : 0x43004300u);
    bool ok = true;
#pragma unroll 1
    for (int b = turn; b < blocks; b += L4_GROUPS) {
      const Fetched now = next;
      if (b + L4_GROUPS < blocks) fetch(b + L4_GROUPS);
      uint32_t w[32];
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const Decoder<T, ST> decode(now.zero[WIDE ? 0 : s], now.scale[WIDE ? 0 : s]);
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
          for (int e = 0; e < 2; ++e)  // inputs 16 s + 4 q + 2 e and the next: nibbles 2 (s % 2) + e of word s / 2
            w[8 * s + 2 * q + e] = decode((s / 2 ? now.codes[q].y : now.codes[q].x) >> (8 * (s % 2) + 4 * e), offset);
      }
      const int ws = b % L4_WEIGHT_STAGES;
      if (b >= L4_WEIGHT_STAGES && !__all_sync(0xffffffffu, mbar_wait(smem_u32(&bar_w_empty[ws]), ((b / L4_WEIGHT_STAGES) & 1u) ^ 1u, abortp))) {
        if (lane == 0) give_up(63);
        ok = false;
        break;
      }
      tc_fence_after();
      l4_store32(tmem + lane_base + S::kWeights + ws * 32, w);
      asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&bar_w_full[ws]));
    }
    if (ok && !__all_sync(0xffffffffu, mbar_wait(smem_u32(&bar_acc), 0u, abortp))) {
      if (lane == 0) give_up(64);
      ok = false;
    }
    // the four warps of a group go on together or not at all
    asm volatile("bar.sync %0, 128;" ::"r"(1 + turn) : "memory");
    if (!*abortp) {
      tc_fence_after();
      const int out = out0 + r;
      const float bias = a.bias && out < a.n ? a.bias[out] : 0.f;
      const float unfold = a.unfold && out < a.n ? a.unfold[out] : 1.f;
      uint8_t* const staging = base_ptr + turn * 8192;  // 32 rows of 128 outputs
      const int outs = min(L4_OUTPUTS, a.n - out0);
      const bool wide = a.n % 8 == 0 && ((uintptr_t)a.y & 15) == 0;
#pragma unroll 1
      for (int c = 0; c < ROWS / (32 * L4_GROUPS); ++c) {
        const int first = turn * (ROWS / L4_GROUPS) + c * 32;
        uint32_t v[32];
        tmem_ld32_nowait(tmem + lane_base + S::kAcc + first, v);
        tmem_ld_wait_for(v);
        if (p.splits > 1) {  // f32 sums, [row][128 outputs], for the cluster
#pragma unroll
          for (int e = 0; e < 32; ++e) *(uint32_t*)(base_ptr + (first + e) * 512 + r * 4) = v[e];
          continue;
        }
#pragma unroll
        for (int e = 0; e < 32; ++e) *(T*)(staging + e * 256 + r * 2) = from_f32<T>(__uint_as_float(v[e]) * unfold + bias);
        asm volatile("bar.sync %0, 128;" ::"r"(1 + turn) : "memory");
        const int i = (int)threadIdx.x & 127;
        if (wide) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int row = e * 8 + i / 16, col = i % 16 * 8;
            if (row0 + first + row < a.rows && col < outs) *(uint4*)((T*)a.y + (row0 + first + row) * a.n + out0 + col) = *(const uint4*)(staging + row * 256 + col * 2);
          }
        } else if (i < outs) {
#pragma unroll 4
          for (int row = 0; row < 32; ++row)
            if (row0 + first + row < a.rows) ((T*)a.y)[(row0 + first + row) * a.n + out0 + i] = *(const T*)(staging + row * 256 + i * 2);
        }
        asm volatile("bar.sync %0, 128;" ::"r"(1 + turn) : "memory");
      }
    }
  }

  // ---------------- teardown ----------------
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (abort_flag && threadIdx.x == 0) {
    // give copies that may still be in flight time to land before the block's shared memory goes away
    const long long start = clock64();
    while (clock64() - start < 2000000LL) {
    }
  }
  __syncthreads();
  // In front of the meeting below: on another stream a cluster of the small-product kernel may hold the columns that a block of this
  // one's waits for while it waits for these.
  if (warp == 4 * L4_GROUPS) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base_slot), "r"(512) : "memory");

  // ---------------- a cluster's sums, in the order of the inputs: every block has its share of the rows ----------------
  if (p.splits > 1) {
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    const int outs = min(L4_OUTPUTS, a.n - out0);
    const bool wide = a.n % 4 == 0 && ((uintptr_t)a.y & 7) == 0;
    for (int i = threadIdx.x; i < ROWS / p.splits * 32; i += L4_THREADS) {
      const int row = split + i / 32 * p.splits, col = i % 32 * 4;
      if (row0 + row >= a.rows || col >= outs) continue;
      float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int c = 0; c < p.splits; ++c) {
        const float4 v = *(const float4*)(cluster.map_shared_rank(base_ptr, c) + row * 512 + col * 4);
        sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
      }
      T out[4];
      const float v[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float y = a.unfold && col + e < outs ? v[e] * a.unfold[out0 + col + e] : v[e];
        out[e] = from_f32<T>(a.bias && col + e < outs ? y + a.bias[out0 + col + e] : y);
      }
      T* const to = (T*)a.y + (row0 + row) * a.n + out0 + col;
      if (wide) *(uint2*)to = *(const uint2*)out;
      else
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (col + e < outs) to[e] = out[e];
    }
    cluster.sync();
  }
}

// Rows whose length is no multiple of 16 bytes, once more with a stride that is one: 16 bytes a thread.
__global__ void __launch_bounds__(256) linear4_pad_rows(const uint16_t* x, uint16_t* padded, int rows, int k, int stride) {
  pdl_enter();
  const int pieces = stride / 8;
  for (int row = blockIdx.x; row < rows; row += gridDim.x) {
    const uint16_t* const src = x + (int64_t)row * k;
    for (int i = threadIdx.x; i < pieces; i += 256) {
      uint32_t w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int at = i * 8 + e * 2;
        w[e] = (at < k ? src[at] : 0u) | (at + 1 < k ? (uint32_t)src[at + 1] : 0u) << 16;
      }
      *(uint4*)(padded + (int64_t)row * stride + i * 8) = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
}

}  // namespace umma

using namespace umma;

namespace {

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn tiled_encoder() {
  static std::once_flag once;
  static EncodeTiledFn fn = nullptr;
  std::call_once(once, [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult qr;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &qr) == cudaSuccess && qr == cudaDriverEntryPointSuccess) fn = (EncodeTiledFn)f;
    (void)cudaGetLastError();
  });
  return fn;
}

template <typename T, int ROWS, typename ST, bool WIDE>
void launch_prompt(const Linear4& a, cudaStream_t s) {
  using S = Linear4Shape<ROWS>;
  static std::mutex mu;
  static bool have[64] = {};
  int device = 0;
  OXB_CUDA(cudaGetDevice(&device));
  {
    std::lock_guard<std::mutex> lock(mu);
    if (device < 0 || device >= 64 || !have[device]) {
      OXB_CUDA(cudaFuncSetAttribute(umma_linear4_kernel<T, ROWS, ST, WIDE>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)S::kSmem));
      if (device >= 0 && device < 64) have[device] = true;
    }
  }
  Linear4Params p{};
  p.a = a;
  p.blocks = (a.k + L4_K - 1) / L4_K;
  while ((1 << p.shift) < a.group) ++p.shift;
  const void* x = a.x;
  int64_t stride = a.k;
  if (a.workspace) {
    stride = (a.k + 7) / 8 * 8;
    launch(linear4_pad_rows, dim3((unsigned)std::min<int64_t>(a.rows, kDependentBlocks)), dim3(256), 0, s, (const uint16_t*)a.x, (uint16_t*)a.workspace, (int)a.rows, a.k, (int)stride);
    x = a.workspace;
  }
  const cuuint64_t dims[2] = {(cuuint64_t)a.k, (cuuint64_t)a.rows}, strides[1] = {(cuuint64_t)stride * 2};
  const cuuint32_t box[2] = {L4_K, ROWS}, steps[2] = {1, 1};
  EncodeTiledFn encode = tiled_encoder();
  if (!encode || encode(&p.x, a.dt == DT::F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(x), dims, strides, box, steps,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
    OXB_FAIL("MatMulNBits: the driver refused the tensor map of x");
  // kind::f16: f32 accumulator, A (from tensor memory) and B in x's type, both K-major, 128 x ROWS
  const uint32_t type = a.dt == DT::F16 ? 0u : 1u;
  p.idesc = (1u << 4) | (type << 7) | (type << 10) | (((uint32_t)ROWS >> 3) << 17) | ((128u >> 4) << 24);
  const int64_t tiles = ceil_div(a.n, L4_OUTPUTS) * ceil_div(a.rows, ROWS);
  if (tiles > 0x7fffffff / 8 || a.rows > 0x7fffffff) OXB_FAIL("MatMulNBits: %lld rows", (long long)a.rows);
  // Where the tiles leave SMs idle, the inputs of each are split over a cluster, four blocks of 64 at least: 256 rows by
  // 4096x4096 27.2 -> 14.6 us, by 8192x4096 49.4 -> 19.7, 64 rows by 4096x4096 21.7 -> 10.6, by 1024x4096 8.2 -> 8.3.  An eighth
  // of the SMs is left out of the count, since clusters do not fill every group of SMs: 144 blocks in fours took two turns.
  p.splits = 1;
  while (p.splits < 8 && tiles * p.splits * 2 <= device_sms() * 7 / 8 && p.blocks >= 4 * p.splits * 2) p.splits *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(tiles * p.splits));
  cfg.blockDim = dim3(L4_THREADS);
  cfg.dynamicSmemBytes = S::kSmem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = p.splits;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.splits > 1 ? 2 : 1;
  OXB_CUDA(cudaLaunchKernelEx(&cfg, umma_linear4_kernel<T, ROWS, ST, WIDE>, p));
}

template <typename T, int ROWS, typename ST>
void launch_prompt(const Linear4& a, cudaStream_t s) { a.group >= L4_K ? launch_prompt<T, ROWS, ST, true>(a, s) : launch_prompt<T, ROWS, ST, false>(a, s); }
template <typename T>
void launch_prompt(const Linear4& a, cudaStream_t s) {
  if (a.rows <= 128) a.scales_f16 ? launch_prompt<T, 128, __half>(a, s) : launch_prompt<T, 128, float>(a, s);
  else a.scales_f16 ? launch_prompt<T, 256, __half>(a, s) : launch_prompt<T, 256, float>(a, s);
}

}  // namespace

// A weight (code - zero) * scale is normal in x's type from its least normal number up, and finite up to its largest; products with
// f16 scales of any size are exact below f16's normal numbers.  An output that has scales outside of that gets the power of two
// that puts its largest scale at 2^11 (f16: 15 times it still fits) or 1 (bf16), from where 25 (126) powers of two lie above the
// least normal number.
bool linear4_folds(const Linear4& a, const float* scales, bool zero_points, std::vector<int>* folds) {
  const bool f16 = a.dt == DT::F16;
  const double most = f16 ? 65504.0 : 0x1.fep127, least = f16 ? 0x1p-14 : 0x1p-126, reach = zero_points ? 15.0 : 8.0;
  std::vector<int> out((size_t)a.n, 0);
  bool any = false;
  for (int64_t n = 0; n < a.n; ++n) {
    double high = 0.0, low = HUGE_VAL;
    for (int g = 0; g < a.groups; ++g) {
      const double v = std::fabs((double)scales[n * a.groups + g]);
      if (!std::isfinite(v)) return false;  // it is the sum of its group that is multiplied by it
      high = std::max(high, v);
      if (v > 0.0) low = std::min(low, v);
    }
    if (high * reach <= most && (low >= least || a.scales_f16)) continue;
    const int fold = (f16 ? 11 : 0) - std::ilogb(high);
    if (std::ldexp(low, fold) < least) return false;
    out[n] = fold;
    any = true;
  }
  if (any) folds->swap(out);
  return true;
}

// Rows that TMA does not take as they lie (their length no multiple of 16 bytes) are copied.
size_t linear4_workspace(const Linear4& a) { return linear4_many_rows(a) && a.k % 8 != 0 ? (size_t)a.rows * ((a.k + 7) / 8 * 8) * 2 : 0; }

void linear4_prompt(const Linear4& a, cudaStream_t s) { a.dt == DT::F16 ? launch_prompt<__half>(a, s) : launch_prompt<__nv_bfloat16>(a, s); }

}  // namespace k
}  // namespace oxb
