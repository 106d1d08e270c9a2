// Causal attention of packed sequences' new rows over the pages of a cache.
//
// out[i] = sum_j p_j v_j / sum_j p_j with p_j = exp(scale (q_i . k_j) - max), over the positions j up to the row's own.  The
// query heads that share a key head are rows beside one another ("packed rows": row r of a sequence is head r % group of
// its new token r / group), so that a tile of keys is read once for all of them.
//
// Sequences of few packed rows (single tokens of a decoding step) are bound by the bytes of their keys and values: this
// file's kernel streams those, at 5.5 TB/s over 64 streams of up to 8100 tokens (196 to 202 us, by the GPU) and 5.2 over one of
// 131000 (103 us, 10 of them beginning and joining), 32 heads on 8 key heads of 128.  Sequences of many are bound by the products
// and run on tcgen05 (umma_prompt.cu).  Each kernel finds its own sequences in the row bounds and skips the others.
#include <algorithm>
#include <mutex>

#include "decoder_device.cuh"

namespace oxb {
namespace k {

namespace {

constexpr int kRows = 16;       // packed rows of a work unit: one m16n8k16 fragment
constexpr int kPiece = 16;      // keys that a warp takes at a time; a page holds a whole number of them
constexpr int kShortRows = 64;  // packed rows of a sequence up to which it is streamed: its keys are read once for every 16 of them
// Pieces that beginning and ending a unit costs, and steps that a warp takes at least, below which joining the parts costs more
// than the keys.  4 short streams (12 heads of 64, 700 tokens) with at least 4 / 8 / 16 steps 15.7 / 19.7 / 27.8 us; 64 streams
// of up to 8100 tokens with 2 / 4 / 8 pieces 195.9 / 196.5 / 197.9.
constexpr int kBegin = 2, kLeast = 4;
// A probability is 2^(score slope - maximum slope), one multiplication and addition with the rounded product of the maximum, whose
// error (2^-24 of it) is a factor of the whole row.  Where the product is above this, parts whose maxima differ would no longer fit
// together (2^-14 here; from 2^28 on powers of two overflow): there the maximum is taken off the scores first.
constexpr float kFar = 1024.f;

// Lanes of a head in shared memory (zeros behind its own), warps of a block and stages of a warp's ring.  A warp streams a piece
// of keys and one of values a stage through cp.async and keeps its own maximum, sum and accumulator.
template <int KD>
struct Shape {
  static constexpr int kWarps = KD == 256 ? 4 : 8;
  static constexpr int kStages = KD == 64 ? 5 : 3;
  static constexpr int kStage = 2 * kPiece * KD * 2;
  static constexpr int kRing = kStages * kStage;
  static constexpr size_t kSmem = (size_t)kWarps * kRing;
  // floats that a part of a unit leaves in the workspace: the accumulator in the order of its fragments, maximum and sum of
  // each row
  static constexpr size_t kPart = (size_t)kRows * KD + 2 * kRows;
};

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

// in 32 bits where both fit, as they do for all but absurd sizes: the division of 64-bit numbers is a hundred instructions
__device__ __forceinline__ long long quotient(long long x, long long y) {
  return ((unsigned long long)(x | y) >> 32) ? x / y : (long long)((unsigned)x / (unsigned)y);
}
__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// log2 of what the largest probability of a row is written as.  Probabilities are rounded to 16 bits for their product with the
// values, and the many small ones of a long past may be all that an output is made of: in f16, whose normal numbers end at 2^-14,
// the largest is 2^15, so that they go down to 2^-29 of it; bf16 has f32's range.  The sums are as much larger and take it out.
template <typename T>
constexpr float kLift = 0.f;
template <>
constexpr float kLift<__half> = 15.f;
__device__ __forceinline__ uint32_t pack16(float lo, float hi, __half*) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *(const uint32_t*)&h;
}
__device__ __forceinline__ uint32_t pack16(float lo, float hi, __nv_bfloat16*) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *(const uint32_t*)&h;
}

// A unit of work (16 packed rows of a sequence for one key head) as a warp goes through its keys.
struct Unit {
  int b, index, units;                   // sequence, unit of it and how many it has
  int pieces;                            // of 16 keys, at least one: a unit that sees nothing writes its zeros
  int first, rows, length, kv, row0;     // of the sequence; key head and first packed row of the unit
  bool bad;
};

// A warp's work is a run of steps out of all units' laid end to end (sequence, key head, 16 packed rows; a unit has kBegin
// steps and one for every piece of 16 keys; the units of a sequence have the same number), and the runs of a block's warps lie
// side by side.  A unit that lies in one warp's run is written by it.  Of any other the warps leave parts in the workspace;
// their block joins them when its warps are done, and the parts of blocks are joined by the block that brings the last one.
// Parts are joined in the order of the keys, whoever does it.
//
// Warps of a block share nothing until then: no barrier stands in their loops, and a warp's loads run on from one unit into the
// next.  `slope` is scale * log2(e) without its sign, `flip` the sign to give the queries' lanes, `mute` a scale of 0.
template <typename T, int KD>
__global__ void __launch_bounds__(Shape<KD>::kWarps * 32, 1) paged_attention_short(PagedAttention a, int most_rows, float slope, uint32_t flip, bool mute) {
  using S = Shape<KD>;
  constexpr int W = S::kWarps, THREADS = W * 32, CH = KD / 8;  // CH: 16-byte pieces of a head
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ long long scan[W];
  struct Part {
    int valid;  // 1: fragments in the workspace, 2: in shared memory
    int c0, c1, first, rows, kv, row0;
  };
  __shared__ Part parts[W][2];  // [0] of a unit that began in an earlier warp, [1] of one that goes on in the next
  __shared__ float part_max[W * 2 * kRows], part_sum[W * 2 * kRows];  // of those parts: rows
  __shared__ int last_part[W + 1];
  pdl_enter();
  const int tid = threadIdx.x, warp = tid / 32, lane = tid & 31, quad = lane & 3, group = a.heads / a.kv_heads, B = a.t.sequences;
  long long* const ends = (long long*)(smem + S::kSmem);  // steps of sequences 0 .. b
  if (tid < 2 * W) parts[tid / 2][tid & 1].valid = 0;

  // ---- steps of each sequence, summed up ----
  auto units_of = [&](const Sequence& q) {
    const long long rows = (long long)q.rows * group;
    return rows > 0 && rows <= most_rows ? a.kv_heads * (int)((rows + kRows - 1) / kRows) : 0;
  };
  auto pieces_of = [&](const Sequence& q) { return max(1, (q.length + kPiece - 1) / kPiece); };
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
      sum = (long long)units_of(q) * (pieces_of(q) + kBegin);
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
  const int warps = (int)gridDim.x * W, me = (int)blockIdx.x * W + warp;
  const long long per = max((long long)kLeast, quotient(total + warps - 1, warps));
  const long long begin = me * per, stop = min(total, begin + per);
  float* const slots = (float*)a.workspace;  // a part to a warp, then two to a block
  float* const block_slots = slots + (size_t)warps * S::kPart;
  int* const counters = (int*)(block_slots + (size_t)gridDim.x * 2 * S::kPart);

  auto load_unit = [&](int b, int index) {
    Unit u;
    const Sequence q = sequence_of(a.t, b, &u.bad);
    const int row_tiles = (q.rows * group + kRows - 1) / kRows;
    u.b = b, u.index = index, u.units = a.kv_heads * row_tiles;
    u.pieces = pieces_of(q);
    u.first = q.first, u.rows = q.rows, u.length = q.length;
    u.kv = index / row_tiles, u.row0 = index % row_tiles * kRows;  // the row tiles of a key head lie side by side
    return u;
  };
  auto next_unit = [&](const Unit& u) {  // there is one: the run goes on
    if (u.index + 1 < u.units) return load_unit(u.b, u.index + 1);
    int b = u.b + 1;
    while (b < B - 1 && ends[b] == ends[b - 1]) ++b;
    return load_unit(b, 0);
  };

  float acc[KD / 8][4], most[2], sum[2];
  bool pending = false;  // the last unit's part is still in the registers
  if (begin < stop) {
    // ---- where the run begins ----
    int b = 0;
    for (int hi = B - 1; b < hi;) {
      const int mid = (b + hi) / 2;
      if (ends[mid] > begin) hi = mid;
      else b = mid + 1;
    }
    const long long seq_start = b > 0 ? ends[b - 1] : 0;
    Unit u = load_unit(b, 0);
    {
      const int index = (int)quotient(begin - seq_start, u.pieces + kBegin);
      u = load_unit(b, index);
    }
    long long unit_at = seq_start + (long long)u.index * (u.pieces + kBegin);  // the unit's first step
    int piece = (int)max(0LL, begin - unit_at - kBegin);
    // pieces of this run from here on
    int left = 0;
    {
      // count them unit by unit (a run holds few units, or short ones)
      long long at = begin;
      Unit v = u;
      long long v_at = unit_at;
      while (true) {
        const long long end = min(stop, v_at + kBegin + v.pieces);
        left += (int)max(0LL, end - max(at, v_at + kBegin));
        at = end;
        if (end == stop) break;
        v_at = end;
        v = next_unit(v);
      }
    }
    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem) + warp * S::kRing;

    // ---- the loads run ahead of the products, with a place of their own in the run ----
    Unit f = u;
    int f_piece = piece, f_left = left;
    int f_page_at = f_piece * kPiece / a.t.page, f_row = f_piece * kPiece % a.t.page;  // entry of the page table, row of the page
    auto page_of = [&]() -> int {
      if (f_left == 0 || f_piece * kPiece >= f.length) return -1;
      const int page = a.t.page_table[(int64_t)f.b * a.t.max_pages + f_page_at];
      if (page >= 0 && page < a.t.pages) return page;
      if (lane == 0 && !f.bad) report(a.err, kErrPage);  // of a cut length the table says nothing
      return -1;
    };
    constexpr int RPI = 32 / CH > 0 ? 32 / CH : 1;  // rows that the warp's lanes fetch with one instruction
    const int lane_row = lane / CH, lane_col = lane % CH;
    const uint32_t lane_dst = lane_row * (KD * 2) + ((lane_col ^ lane_row) << 4);
    const int64_t lane_src = (int64_t)lane_row * a.kv_heads * a.size + lane_col * 8, step = (int64_t)RPI * a.kv_heads * a.size;
    int stage_in = 0;
    auto fetch = [&](int page) {  // keys and values behind the sequence, and lanes behind the head, are zeros
      const uint32_t dst = ring + stage_in * S::kStage + lane_dst;
      const int64_t row = ((int64_t)max(page, 0) * a.t.page + f_row) * a.kv_heads + f.kv;
      const T *k = (const T*)a.key_cache + row * a.size + lane_src, *v = (const T*)a.value_cache + row * a.size + lane_src;
      if (page >= 0 && (f_piece + 1) * kPiece <= f.length && a.size == KD) {
#pragma unroll
        for (int e = 0; e < kPiece / RPI; ++e) {
          const uint32_t to = (dst ^ (uint32_t)((e * RPI & 7) << 4)) + e * RPI * (KD * 2);
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(k) : "memory");
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + kPiece * KD * 2), "l"(v) : "memory");
          k += step, v += step;
        }
      } else {
#pragma unroll
        for (int e = 0; e < kPiece / RPI; ++e) {
          const uint32_t to = (dst ^ (uint32_t)((e * RPI & 7) << 4)) + e * RPI * (KD * 2);
          const bool valid = page >= 0 && f_piece * kPiece + e * RPI + lane_row < f.length && lane_col * 8 < a.size;
          cp_async16(to, valid ? k : (const T*)a.key_cache, valid);
          cp_async16(to + kPiece * KD * 2, valid ? v : (const T*)a.value_cache, valid);
          k += step, v += step;
        }
      }
      if (++stage_in == S::kStages) stage_in = 0;
    };
    auto advance = [&]() {  // to the piece that is fetched next
      --f_left;
      f_row += kPiece;
      if (f_row == a.t.page) f_row = 0, ++f_page_at;
      if (++f_piece == f.pieces && f_left > 0) {
        f = next_unit(f);
        f_piece = f_page_at = f_row = 0;
      }
    };
    int ahead = page_of();
#pragma unroll 1
    for (int i = 0; i < S::kStages - 1; ++i) {
      if (f_left > 0) {
        fetch(ahead);
        advance();
        ahead = page_of();
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    }

    int stage = 0;
#pragma unroll 1
    while (left > 0) {
      // ---- the queries' fragments: rows lane / 4 and lane / 4 + 8 of the 16 ----
      const int rows = u.rows * group;
      uint32_t qf[KD / 16][4];
      int limit[2];
      const T* src[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {  // rows behind the last are copies of it that nobody stores
        const int r = min(u.row0 + lane / 4 + 8 * h, rows - 1), token = r / group;
        limit[h] = max(0, u.length - u.rows + token + 1);
        src[h] = (const T*)a.q + ((int64_t)(u.first + token) * a.heads + u.kv * group + (r - token * group)) * a.size + quad * 2;
      }
      if (a.size == KD && !mute) {
#pragma unroll
        for (int k = 0; k < KD / 16; ++k)
#pragma unroll
          for (int e = 0; e < 4; ++e) qf[k][e] = *(const uint32_t*)(src[e & 1] + k * 16 + e / 2 * 8);
      } else {
#pragma unroll
        for (int k = 0; k < KD / 16; ++k)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int d = k * 16 + e / 2 * 8;
            const uint32_t v = *(const uint32_t*)(src[e & 1] + (d < a.size ? d : 0));
            qf[k][e] = d < a.size && !mute ? v : 0u;
          }
      }
      if (flip)
#pragma unroll
        for (int k = 0; k < KD / 16; ++k)
#pragma unroll
          for (int e = 0; e < 4; ++e) qf[k][e] ^= flip;
      most[0] = most[1] = -INFINITY, sum[0] = sum[1] = 0.f;
      float bias[2] = {0.f, 0.f};  // what is taken off scaled scores
      bool far = false;            // a maximum is far from 0: it is taken off the scores before they are scaled
#pragma unroll
      for (int n = 0; n < KD / 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[n][e] = 0.f;

      const int piece0 = piece, piece1 = min(u.pieces, piece + left);
#pragma unroll 1
      for (; piece < piece1; ++piece) {
        asm volatile("cp.async.wait_group %0;" ::"n"(S::kStages - 2) : "memory");
        __syncwarp();  // every lane's pieces have landed, and every lane is done with the stage that is filled next
        if (f_left > 0) {
          fetch(ahead);
          advance();
          ahead = page_of();
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        const uint32_t keys = ring + stage * S::kStage, values = keys + kPiece * KD * 2;
        if (++stage == S::kStages) stage = 0;

        float s[2][4] = {};
#pragma unroll
        for (int k = 0; k < KD / 16; ++k) {
          uint32_t m[4];
          const int r = (lane & 7) + ((lane >> 4) << 3), c = 2 * k + ((lane >> 3) & 1);
          ldmatrix4(m, keys + r * (KD * 2) + ((c ^ (r & 7)) << 4));
          mma16816<T>(s[0], qf[k], m[0], m[1]);
          mma16816<T>(s[1], qf[k], m[2], m[3]);
        }
        if (piece * kPiece + kPiece > min(limit[0], limit[1])) {
          const int key = piece * kPiece + quad * 2;
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (key + n * 8 + (e & 1) >= limit[e / 2]) s[n][e] = -INFINITY;
        }
        float top[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          top[h] = fmaxf(fmaxf(s[0][2 * h], s[0][2 * h + 1]), fmaxf(s[1][2 * h], s[1][2 * h + 1]));
          top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 1));
          top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 2));
          top[h] = fmaxf(top[h], most[h]);
        }
        if (far || __any_sync(0xffffffffu, top[0] > most[0] || top[1] > most[1])) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float keep = most[h] == -INFINITY ? 0.f : exp2_approx((most[h] - top[h]) * slope);
            most[h] = top[h];
            sum[h] *= keep;
#pragma unroll
            for (int n = 0; n < KD / 8; ++n) acc[n][2 * h] *= keep, acc[n][2 * h + 1] *= keep;
            bias[h] = most[h] == -INFINITY ? 0.f : fmaf(most[h], slope, -kLift<T>);
          }
          far = __any_sync(0xffffffffu, fabsf(bias[0]) > kFar || fabsf(bias[1]) > kFar);
          if (far) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              if (most[h] == -INFINITY) continue;  // so are the scores
              bias[h] = -kLift<T>;
#pragma unroll
              for (int n = 0; n < 2; ++n) s[n][2 * h] -= most[h], s[n][2 * h + 1] -= most[h];
            }
          }
        }
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
          uint32_t m[4];
          const int r = lane & 15, c = 2 * n + (lane >> 4);
          ldmatrix4_trans(m, values + r * (KD * 2) + ((c ^ (r & 7)) << 4));
          mma16816<T>(acc[2 * n], p, m[0], m[1]);
          mma16816<T>(acc[2 * n + 1], p, m[2], m[3]);
        }
      }
      left -= piece1 - piece0;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 1);
        sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 2);
      }
      // ---- the unit's rows, or this warp's part of them ----
      const int c0 = (int)quotient(unit_at + kBegin, per), c1 = (int)quotient(unit_at + kBegin + u.pieces - 1, per);
      if (c0 == c1) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int row = u.row0 + lane / 4 + 8 * h;
          const float inv = sum[h] > 0.f ? 1.f / sum[h] : sum[h] == 0.f ? 0.f : sum[h];  // NaN where a key was
          T* const to = (T*)a.out + ((int64_t)(u.first + row / group) * a.heads + u.kv * group + row % group) * a.size;
          if (row < rows)
#pragma unroll
            for (int n = 0; n < KD / 8; ++n)
              if (n * 8 < a.size) *(uint32_t*)(to + n * 8 + quad * 2) = pack16(acc[n][2 * h] * inv, acc[n][2 * h + 1] * inv, (T*)nullptr);
        }
      } else {
        const int which = piece0 == 0 ? 1 : 0;
        if (left > 0) {  // the last one's fragments stay in the registers until the rings are free
          float* const slot = slots + (size_t)me * S::kPart;
#pragma unroll
          for (int n = 0; n < KD / 8; ++n) ((float4*)slot)[n * 32 + lane] = make_float4(acc[n][0], acc[n][1], acc[n][2], acc[n][3]);
        } else {
          pending = true;
        }
        if (quad == 0)
#pragma unroll
          for (int h = 0; h < 2; ++h) part_max[(warp * 2 + which) * kRows + lane / 4 + 8 * h] = most[h], part_sum[(warp * 2 + which) * kRows + lane / 4 + 8 * h] = sum[h];
        if (lane == 0) parts[warp][which] = Part{left > 0 ? 1 : 2, c0, c1, u.first, u.rows, u.kv, u.row0};
      }
      if (left > 0) {
        unit_at += u.pieces + kBegin;
        u = next_unit(u);
        piece = 0;
      }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
  }
  __threadfence();
  __syncthreads();
  float* const held = (float*)smem;  // [warp]: the parts that were still in registers, where the rings were
  if (pending)
#pragma unroll
    for (int n = 0; n < KD / 8; ++n) ((float4*)(held + (size_t)warp * kRows * KD))[n * 32 + lane] = make_float4(acc[n][0], acc[n][1], acc[n][2], acc[n][3]);
  __syncthreads();

  // ---- the parts that this block's warps left, all units' at once ----
  // Rows g and g + 8 of fragment `i` (n * 32 + lane) out of the parts p0 .. p1: `at(p, i)` is a part's fragment, `max_of`
  // and `sum_of` (p, row) are what its rows have.  Relative to the largest maximum: v, and maxima and sums in m and w.
  auto join = [&](auto at, auto max_of, auto sum_of, int p0, int p1, int i, float (&v)[4], float (&m)[2], float (&w)[2]) {
    const int g = (i & 31) / 4;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      m[h] = -INFINITY, w[h] = 0.f;
      for (int p = p0; p <= p1; ++p) m[h] = fmaxf(m[h], max_of(p, g + 8 * h));
    }
    v[0] = v[1] = v[2] = v[3] = 0.f;
    for (int p = p0; p <= p1; p += 8) {  // eight loads in flight
      float4 x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = p + e <= p1 ? at(p + e, i) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (p + e > p1) break;
        float keep[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float top = max_of(p + e, g + 8 * h);
          keep[h] = top == -INFINITY ? 0.f : exp2_approx((top - m[h]) * slope);
          w[h] += sum_of(p + e, g + 8 * h) * keep[h];
        }
        v[0] += x[e].x * keep[0], v[1] += x[e].y * keep[0], v[2] += x[e].z * keep[1], v[3] += x[e].w * keep[1];
      }
    }
  };
  auto finish = [&](const Part& t, int i, const float (&v)[4], const float (&w)[2]) {
    const int d = i / 32 * 8 + (i & 3) * 2;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int row = t.row0 + (i & 31) / 4 + 8 * h;
      if (row >= t.rows * group || d >= a.size) continue;
      const float inv = w[h] > 0.f ? 1.f / w[h] : w[h] == 0.f ? 0.f : w[h];
      *(uint32_t*)((T*)a.out + ((int64_t)(t.first + row / group) * a.heads + t.kv * group + row % group) * a.size + d) = pack16(v[2 * h] * inv, v[2 * h + 1] * inv, (T*)nullptr);
    }
  };
  // Units by their first warp in this block: number 0 began in an earlier block, number e in warp e - 1.
  constexpr int FRAGMENTS = KD / 8 * 32;
  const int warp0 = (int)blockIdx.x * W;
  auto unit_part = [&](int e) -> const Part& { return e == 0 ? parts[0][0] : parts[e - 1][1]; };
  bool across = false;
  for (int i = tid; i < (W + 1) * FRAGMENTS; i += THREADS) {
    const int e = i / FRAGMENTS, at = i % FRAGMENTS;
    const Part& t = unit_part(e);
    if (!t.valid) continue;
    const int block0 = t.c0 / W;
    auto which = [&](int p) { return p * 2 + (p == t.c0 ? 1 : 0); };  // of a warp's two parts
    float v[4], m[2], w[2];
    auto fragment = [&](int p, int f) {  // a warp that went on to another unit left its part in the workspace
      const int w = p - warp0;
      return parts[w][p == t.c0 ? 1 : 0].valid == 2 ? ((const float4*)(held + (size_t)w * kRows * KD))[f] : __ldcg((const float4*)(slots + (size_t)p * S::kPart) + f);
    };
    join(fragment, [&](int p, int row) { return part_max[(which(p) - 2 * warp0) * kRows + row]; },
         [&](int p, int row) { return part_sum[(which(p) - 2 * warp0) * kRows + row]; }, max(t.c0, warp0), min(t.c1, warp0 + W - 1), at, v, m, w);
    if (block0 == t.c1 / W) {
      finish(t, at, v, w);
    } else {
      float* const mine = block_slots + ((size_t)blockIdx.x * 2 + (block0 == (int)blockIdx.x ? 1 : 0)) * S::kPart;
      ((float4*)mine)[at] = make_float4(v[0], v[1], v[2], v[3]);
      if (at < 32 && (at & 3) == 0)
#pragma unroll
        for (int h = 0; h < 2; ++h) mine[kRows * KD + at / 4 + 8 * h] = m[h], mine[kRows * KD + kRows + at / 4 + 8 * h] = w[h];
    }
  }
  for (int e = 0; e <= W; ++e) across = across || (unit_part(e).valid && unit_part(e).c0 / W != unit_part(e).c1 / W);
  if (!across) return;

  // ---- units that other blocks have parts of, at most two: whoever brings the last part joins them ----
  __threadfence();
  __syncthreads();
  if (tid <= W) {
    const Part& t = unit_part(tid);
    const int block0 = t.c0 / W, block1 = t.c1 / W;
    last_part[tid] = 0;
    if (t.valid && block0 != block1) {
      last_part[tid] = atomicAdd(counters + block0, 1) == block1 - block0;
      if (last_part[tid]) counters[block0] = 0;  // nobody else comes: ready for the next launch
    }
  }
  __syncthreads();
  float* const rows_of = (float*)smem;  // maxima, then sums, of every part's rows: where the rings were
  for (int e = 0; e <= W; ++e) {
    if (!last_part[e]) continue;
    __threadfence();
    const Part& t = unit_part(e);
    const int block0 = t.c0 / W, block1 = t.c1 / W;
    auto part = [&](int p) { return block_slots + ((size_t)p * 2 + (p == block0 ? 1 : 0)) * S::kPart; };
    for (int i = tid; i < (block1 - block0 + 1) * 2 * kRows; i += THREADS) rows_of[i] = __ldcg(part(block0 + i / (2 * kRows)) + kRows * KD + i % (2 * kRows));
    __syncthreads();
    for (int i = tid; i < FRAGMENTS; i += THREADS) {
      float v[4], m[2], w[2];
      join([&](int p, int f) { return __ldcg((const float4*)part(p) + f); }, [&](int p, int row) { return rows_of[(p - block0) * 2 * kRows + row]; }, [&](int p, int row) { return rows_of[(p - block0) * 2 * kRows + kRows + row]; }, block0, block1, i,
           v, m, w);
      finish(t, i, v, w);
    }
    __syncthreads();
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
  launch(paged_attention_short<T, KD>, dim3(device_sms()), dim3(Shape<KD>::kWarps * 32), smem, s, a, most_rows, scale * 1.4426950408889634f,
         a.scale < 0.f ? 0x80008000u : 0u, a.scale == 0.f);
}

template <typename T>
void launch_short(const PagedAttention& a, int most_rows, cudaStream_t s) {
  if (a.size <= 64) launch_short<T, 64>(a, most_rows, s);
  else if (a.size <= 128) launch_short<T, 128>(a, most_rows, s);
  else launch_short<T, 256>(a, most_rows, s);
}

template <int KD>
constexpr size_t short_parts() { return ((size_t)Shape<KD>::kWarps + 2) * Shape<KD>::kPart; }  // floats for a block: a part to a warp, and two

size_t short_workspace(const PagedAttention& a) {
  const size_t floats = a.size <= 64 ? short_parts<64>() : a.size <= 128 ? short_parts<128>() : short_parts<256>();
  return align_up((size_t)device_sms() * (floats * sizeof(float) + sizeof(int)), 256);
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
