// Causal attention of packed sequences' new rows over the pages of a cache.
//
// out[i] = sum_j p_j v_j / sum_j p_j with p_j = exp(scale (q_i . k_j) - max), over the positions j up to the row's own.  The
// query heads that share a key head are rows beside one another ("packed rows": row r of a sequence is head r % group of
// its new token r / group), so that a tile of keys is read once for all of them.
//
// Sequences of few packed rows (single tokens of a decoding step) are bound by the bytes of their keys and values: this
// file's kernel streams those.  Sequences of many are bound by the products and run on tcgen05 (umma_prompt.cu).  Each
// kernel finds its own sequences in the row bounds and skips the others.
#include <algorithm>
#include <mutex>

#include "decoder_device.cuh"

namespace oxb {
namespace k {

namespace {

constexpr int kRows = 16;  // packed rows of a work unit: one m16n8k16 fragment

// Lanes of a head in shared memory (zeros behind its own), warps of a block and stages of a warp's ring.  A warp streams 16
// keys and 16 values a stage through cp.async and keeps its own maximum, sum and accumulator: no barrier until a unit ends.
template <int KD>
struct Shape {
  static constexpr int kWarps = KD == 256 ? 4 : 8;
  static constexpr int kStages = KD == 64 ? 5 : 3;
  static constexpr int kStage = 2 * 16 * KD * 2;
  static constexpr int kRing = kStages * kStage;
  static constexpr int kTile = 16 * kWarps;  // keys of a tile: what the warps of a block take in one step
  // floats that a part of a unit leaves in the workspace: accumulator, then maximum and sum of each row; two parts to a
  // block, [0] of a unit that began in an earlier block, [1] of one that goes on in the next
  static constexpr size_t kPart = (size_t)kRows * KD + 2 * kRows;
  static constexpr size_t kSmem = (size_t)kWarps * kRing;
  static_assert(kSmem >= (size_t)kWarps * kRows * KD * 4, "the warps' accumulators meet where the ring was");
};
constexpr int kShortRows = 64;  // packed rows of a sequence up to which it is streamed
constexpr int kMinTiles = 2;  // tiles that a block takes at least: below, joining the parts costs more than the keys

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack16(float lo, float hi, __half*) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *(const uint32_t*)&h;
}
__device__ __forceinline__ uint32_t pack16(float lo, float hi, __nv_bfloat16*) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *(const uint32_t*)&h;
}

// Work of a block: a run of tiles out of all units' tiles laid end to end (sequence, key head, 16 packed rows; the units of
// a sequence have the same number of tiles).  A unit that a run's border cuts leaves its parts in the workspace, and the
// block that brings the last part joins them in the order of the keys, whoever that is: the result does not depend on it.
//
// `slope` is scale * log2(e) without its sign, `flip` the sign to give the queries' lanes, `mute` a scale of 0.
template <typename T, int KD>
__global__ void __launch_bounds__(Shape<KD>::kWarps * 32, 1)
paged_attention_short(PagedAttention a, int most_rows, int min_tiles, float slope, uint32_t flip, bool mute) {
  using S = Shape<KD>;
  constexpr int W = S::kWarps, THREADS = W * 32, CH = KD / 8;  // CH: 16-byte pieces of a head
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ long long scan[W];
  __shared__ float part_max[W][kRows], part_sum[W][kRows];
  __shared__ int last_part;
  pdl_enter();
  const int tid = threadIdx.x, warp = tid / 32, lane = tid & 31, quad = lane & 3, group = a.heads / a.kv_heads, B = a.t.sequences;
  long long* const ends = (long long*)(smem + S::kSmem);  // tiles of sequences 0 .. b

  // ---- tiles of each sequence, summed up ----
  long long total = 0;
  for (int first = 0; first < B; first += THREADS) {
    const int b = first + tid;
    long long sum = 0;
    if (b < B) {
      bool bad;
      const Sequence q = sequence_of(a.t, b, &bad);
      if (blockIdx.x == 0) {
        if (bad) report(a.err, kErrLengths);
        else if (a.max_query > 0 && q.rows > a.max_query) report(a.err, kErrQueryLength);
      }
      const long long rows = (long long)q.rows * group;
      if (rows > 0 && rows <= most_rows)  // a unit without keys has a tile too: it writes the rows' zeros
        sum = (long long)a.kv_heads * ((rows + kRows - 1) / kRows) * max(1, (q.length + S::kTile - 1) / S::kTile);
    }
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const long long up = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += up;
    }
    if (lane == 31) scan[warp] = sum;
    __syncthreads();
    long long base = total;
    for (int w = 0; w < W; ++w) {
      if (w < warp) base += scan[w];
      total += scan[w];
    }
    if (b < B) ends[b] = base + sum;
    __syncthreads();
  }
  // rows behind the last sequence
  for (int64_t i = max(0, a.t.cu_query[B]) * (int64_t)a.heads * a.size / 8 + (int64_t)blockIdx.x * THREADS + tid; i < a.t.tokens * a.heads * a.size / 8; i += (int64_t)gridDim.x * THREADS)
    ((uint4*)a.out)[i] = make_uint4(0, 0, 0, 0);

  const long long per = max((long long)min_tiles, (total + gridDim.x - 1) / gridDim.x);
  long long at = blockIdx.x * per;
  const long long stop = min(total, at + per);
  const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem) + warp * S::kRing;
  while (at < stop) {
    // ---- the unit that tile `at` belongs to ----
    int b = 0;
    for (int hi = B - 1; b < hi;) {
      const int mid = (b + hi) / 2;
      if (ends[mid] > at) hi = mid;
      else b = mid + 1;
    }
    bool bad;
    const Sequence q = sequence_of(a.t, b, &bad);
    const long long seq_start = b > 0 ? ends[b - 1] : 0;
    const int tiles = max(1, (q.length + S::kTile - 1) / S::kTile), rows = q.rows * group, row_tiles = (rows + kRows - 1) / kRows;
    const int unit = (int)((at - seq_start) / tiles), tile0 = (int)((at - seq_start) % tiles);
    const int tile1 = (int)min((long long)tiles, tile0 + (stop - at));
    const int kv = unit / row_tiles, row0 = (unit % row_tiles) * kRows;  // the row tiles of a key head lie side by side
    const int* const pages = a.t.page_table + (int64_t)b * a.t.max_pages;

    // ---- this warp's stream of 16-key pieces: piece i is keys (tile0 * W + warp + i * W) * 16 ... ----
    const int pieces = tile1 - tile0;
    auto key_of = [&](int i) { return ((tile0 + i) * W + warp) * 16; };
    auto page_of = [&](int i) -> int {
      const int key = key_of(i);
      if (i >= pieces || key >= q.length) return -1;
      const int page = pages[key / a.t.page];
      if (page < 0 || page >= a.t.pages) {
        if (lane == 0 && !bad) report(a.err, kErrPage);  // of a cut length the table says nothing
        return -1;
      }
      return page;
    };
    auto fetch = [&](int i, int page) {  // keys and values behind the sequence, and lanes behind the head, are zeros
      const uint32_t dst = ring + (i % S::kStages) * S::kStage;
      const int key = key_of(i);
      const int64_t row = ((int64_t)max(page, 0) * a.t.page + key % a.t.page) * a.kv_heads + kv;
#pragma unroll
      for (int e = 0; e < CH / 2; ++e) {
        const int idx = e * 32 + lane, r = idx / CH, c = idx % CH;
        const bool valid = page >= 0 && key + r < q.length && c * 8 < a.size;
        const int64_t off = valid ? (row + (int64_t)r * a.kv_heads) * a.size + c * 8 : 0;
        const uint32_t to = dst + r * (KD * 2) + ((c ^ (r & 7)) << 4);
        cp_async16(to, (const T*)a.key_cache + off, valid);
        cp_async16(to + 16 * KD * 2, (const T*)a.value_cache + off, valid);
      }
    };
    int ahead = page_of(0);
#pragma unroll
    for (int i = 0; i < S::kStages - 1; ++i) {
      if (i < pieces) fetch(i, ahead);
      asm volatile("cp.async.commit_group;" ::: "memory");
      ahead = page_of(i + 1);
    }

    // ---- the queries' fragments: rows lane / 4 and lane / 4 + 8 of the 16 ----
    uint32_t qf[KD / 16][4];
    int limit[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = row0 + lane / 4 + 8 * h, token = r / group;
      const bool valid = r < rows;
      limit[h] = valid ? max(0, q.length - q.rows + token + 1) : 0;
      const T* src = (const T*)a.q + ((int64_t)(q.first + (valid ? token : 0)) * a.heads + kv * group + (valid ? r % group : 0)) * a.size;
#pragma unroll
      for (int k = 0; k < KD / 16; ++k)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int d = k * 16 + quad * 2 + e * 8;
          qf[k][h + 2 * e] = valid && !mute && d < a.size ? *(const uint32_t*)(src + d) ^ flip : 0u;
        }
    }
    float acc[KD / 8][4], most[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f};
#pragma unroll
    for (int n = 0; n < KD / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[n][e] = 0.f;

    for (int i = 0; i < pieces; ++i) {
      asm volatile("cp.async.wait_group %0;" ::"n"(S::kStages - 2) : "memory");
      __syncwarp();  // every lane's pieces have landed, and every lane is done with the stage that is filled next
      if (i + S::kStages - 1 < pieces) fetch(i + S::kStages - 1, ahead);
      asm volatile("cp.async.commit_group;" ::: "memory");
      ahead = page_of(i + S::kStages);
      const uint32_t keys = ring + (i % S::kStages) * S::kStage, values = keys + 16 * KD * 2;

      float s[2][4] = {};
#pragma unroll
      for (int k = 0; k < KD / 16; ++k) {
        uint32_t f[4];
        const int r = (lane & 7) + ((lane >> 4) << 3), c = 2 * k + ((lane >> 3) & 1);
        ldmatrix4(f, keys + r * (KD * 2) + ((c ^ (r & 7)) << 4));
        mma16816<T>(s[0], qf[k], f[0], f[1]);
        mma16816<T>(s[1], qf[k], f[2], f[3]);
      }
      const int key = key_of(i) + quad * 2;
      float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (key + n * 8 + (e & 1) >= limit[e / 2]) s[n][e] = -INFINITY;
          top[e / 2] = fmaxf(top[e / 2], s[n][e]);
        }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 1));
        top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 2));
        top[h] = fmaxf(top[h], most[h]);
      }
      if (__any_sync(0xffffffffu, top[0] > most[0] || top[1] > most[1])) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float keep = most[h] == -INFINITY ? 0.f : exp2_approx((most[h] - top[h]) * slope);
          most[h] = top[h];
          sum[h] *= keep;
#pragma unroll
          for (int n = 0; n < KD / 8; ++n) acc[n][2 * h] *= keep, acc[n][2 * h + 1] *= keep;
        }
      }
      const float bias[2] = {most[0] == -INFINITY ? 0.f : most[0] * slope, most[1] == -INFINITY ? 0.f : most[1] * slope};
      uint32_t p[4];
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float x = exp2_approx(fmaf(s[n][2 * h], slope, -bias[h])), y = exp2_approx(fmaf(s[n][2 * h + 1], slope, -bias[h]));
          sum[h] += x + y;
          p[2 * n + h] = pack16(x, y, (T*)nullptr);
        }
#pragma unroll
      for (int n = 0; n < KD / 16; ++n) {
        uint32_t f[4];
        const int r = lane & 15, c = 2 * n + (lane >> 4);
        ldmatrix4_trans(f, values + r * (KD * 2) + ((c ^ (r & 7)) << 4));
        mma16816<T>(acc[2 * n], p, f[0], f[1]);
        mma16816<T>(acc[2 * n + 1], p, f[2], f[3]);
      }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 1);
      sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 2);
    }

    // ---- the warps' parts become the block's ----
    if (quad == 0)
#pragma unroll
      for (int h = 0; h < 2; ++h) part_max[warp][lane / 4 + 8 * h] = most[h], part_sum[warp][lane / 4 + 8 * h] = sum[h];
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();  // maxima are there, and all rings have been read
    float* const meet = (float*)smem;  // [warp][row][KD]
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = lane / 4 + 8 * h;
      float all = -INFINITY;
      for (int w = 0; w < W; ++w) all = fmaxf(all, part_max[w][r]);
      const float keep = most[h] == -INFINITY ? 0.f : exp2_approx((most[h] - all) * slope);
#pragma unroll
      for (int n = 0; n < KD / 8; ++n) *(float2*)(meet + ((size_t)warp * kRows + r) * KD + n * 8 + quad * 2) = make_float2(acc[n][2 * h] * keep, acc[n][2 * h + 1] * keep);
    }
    __syncthreads();
    const bool whole = tile0 == 0 && tile1 == tiles;
    const long long unit_start = seq_start + (long long)unit * tiles;
    const int c0 = (int)(unit_start / per), c1 = (int)((unit_start + tiles - 1) / per);
    float* const part = (float*)a.workspace + ((size_t)blockIdx.x * 2 + (tile0 == 0 ? 1 : 0)) * S::kPart;
    auto store = [&](int r, int d, const float (&v)[8], float w) {
      const int row = row0 + r;
      if (row >= rows || d >= a.size) return;
      const float inv = w > 0.f ? 1.f / w : w == 0.f ? 0.f : w;  // w is NaN where a key was
      uint4 o;
      o.x = pack16(v[0] * inv, v[1] * inv, (T*)nullptr), o.y = pack16(v[2] * inv, v[3] * inv, (T*)nullptr);
      o.z = pack16(v[4] * inv, v[5] * inv, (T*)nullptr), o.w = pack16(v[6] * inv, v[7] * inv, (T*)nullptr);
      *(uint4*)((T*)a.out + ((int64_t)(q.first + row / group) * a.heads + kv * group + row % group) * a.size + d) = o;
    };
    for (int idx = tid; idx < kRows * CH; idx += THREADS) {
      const int r = idx / CH, d = idx % CH * 8;
      float all = -INFINITY, w = 0.f, v[8] = {};
      for (int u = 0; u < W; ++u) all = fmaxf(all, part_max[u][r]);
      for (int u = 0; u < W; ++u) {
        if (part_max[u][r] != -INFINITY) w += part_sum[u][r] * exp2_approx((part_max[u][r] - all) * slope);
        const float4 x = *(const float4*)(meet + ((size_t)u * kRows + r) * KD + d), y = *(const float4*)(meet + ((size_t)u * kRows + r) * KD + d + 4);
        v[0] += x.x, v[1] += x.y, v[2] += x.z, v[3] += x.w, v[4] += y.x, v[5] += y.y, v[6] += y.z, v[7] += y.w;
      }
      if (whole) {
        store(r, d, v, w);
      } else {
        *(float4*)(part + r * KD + d) = make_float4(v[0], v[1], v[2], v[3]);
        *(float4*)(part + r * KD + d + 4) = make_float4(v[4], v[5], v[6], v[7]);
        if (d == 0) part[kRows * KD + r] = all, part[kRows * KD + kRows + r] = w;
      }
    }
    if (!whole) {
      int* const counter = (int*)((float*)a.workspace + (size_t)gridDim.x * 2 * S::kPart) + c0;
      __threadfence();
      __syncthreads();
      if (tid == 0) {
        last_part = atomicAdd(counter, 1) == c1 - c0;
        if (last_part) *counter = 0;  // nobody else comes: ready for the next launch
      }
      __syncthreads();
      if (last_part) {
        __threadfence();
        auto part_of = [&](int c) { return (const float*)a.workspace + ((size_t)c * 2 + (c == c0 ? 1 : 0)) * S::kPart; };
        for (int idx = tid; idx < kRows * CH; idx += THREADS) {
          const int r = idx / CH, d = idx % CH * 8;
          float all = -INFINITY, w = 0.f, v[8] = {};
          for (int c = c0; c <= c1; ++c) all = fmaxf(all, __ldcg(part_of(c) + kRows * KD + r));
          for (int c = c0; c <= c1; ++c) {
            const float* src = part_of(c);
            const float m = __ldcg(src + kRows * KD + r);
            if (m == -INFINITY) continue;
            const float keep = exp2_approx((m - all) * slope);
            w += __ldcg(src + kRows * KD + kRows + r) * keep;
            const float4 x = __ldcg((const float4*)(src + r * KD + d)), y = __ldcg((const float4*)(src + r * KD + d + 4));
            v[0] += x.x * keep, v[1] += x.y * keep, v[2] += x.z * keep, v[3] += x.w * keep;
            v[4] += y.x * keep, v[5] += y.y * keep, v[6] += y.z * keep, v[7] += y.w * keep;
          }
          store(r, d, v, w);
        }
      }
    }
    __syncthreads();  // the ring and the shared words are free again
    at += pieces;
  }
}

template <typename T, int KD>
void launch_short(const PagedAttention& a, int most_rows, cudaStream_t s) {
  const size_t smem = Shape<KD>::kSmem + (size_t)a.t.sequences * sizeof(long long);
  static std::mutex mu;
  static size_t have[64] = {};
  int device = 0;
  OXB_CUDA(cudaGetDevice(&device));
  {
    std::lock_guard<std::mutex> lock(mu);
    if (device < 0 || device >= 64 || have[device] < smem) {
      OXB_CUDA(cudaFuncSetAttribute(paged_attention_short<T, KD>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
      if (device >= 0 && device < 64) have[device] = smem;
    }
  }
  const float scale = a.scale == 0.f ? 1.f : fabsf(a.scale);
  launch(paged_attention_short<T, KD>, dim3(device_sms()), dim3(Shape<KD>::kWarps * 32), smem, s, a, most_rows, kMinTiles, scale * 1.4426950408889634f,
         a.scale < 0.f ? 0x80008000u : 0u, a.scale == 0.f);
}

template <typename T>
void launch_short(const PagedAttention& a, int most_rows, cudaStream_t s) {
  if (a.size <= 64) launch_short<T, 64>(a, most_rows, s);
  else if (a.size <= 128) launch_short<T, 128>(a, most_rows, s);
  else launch_short<T, 256>(a, most_rows, s);
}

size_t short_workspace(const PagedAttention& a) {
  const size_t floats = a.size <= 64 ? Shape<64>::kPart : a.size <= 128 ? Shape<128>::kPart : Shape<256>::kPart;
  return align_up((size_t)device_sms() * (2 * floats * sizeof(float) + sizeof(int)), 256);
}

// Is there a call in which some sequence has more than kShortRows packed rows and tcgen05 takes those?
bool has_prompts(const PagedAttention& a) {
  const int64_t longest = a.max_query > 0 ? a.max_query : a.t.tokens;
  return longest * (a.heads / a.kv_heads) > kShortRows && paged_attention_prompts_fit(a);
}

}  // namespace

int device_sms() {
  static const int sms = [] {
    int n = 0, device = 0;
    if (cudaGetDevice(&device) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device) != cudaSuccess) (void)cudaGetLastError();
    return n > 0 ? n : 148;
  }();
  return sms;
}

size_t paged_attention_workspace(const PagedAttention& a) { return short_workspace(a) + (has_prompts(a) ? paged_attention_prompts_workspace(a) : 0); }

void paged_attention(const PagedAttention& a, cudaStream_t s) {
  if (a.t.tokens == 0) return;
  const bool prompts = has_prompts(a);
  // a head that is too wide for tensor memory, or has more query heads than a tile has rows: the streaming kernel takes all rows
  const int most_rows = prompts || paged_attention_prompts_fit(a) ? kShortRows : 0x7fffffff;
  if (a.dt == DT::F16) launch_short<__half>(a, most_rows, s);
  else launch_short<__nv_bfloat16>(a, most_rows, s);
  if (prompts) paged_attention_prompts(a, kShortRows + 1, (uint8_t*)a.workspace + short_workspace(a), s);
}

}  // namespace k
}  // namespace oxb
