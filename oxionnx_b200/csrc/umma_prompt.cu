// Causal attention of many packed rows over the pages of a cache, on tcgen05: scores and output never leave the SM.
//
// A block takes 256 packed rows (two tiles of 128) of one key head and walks its keys 128 at a time.  Scores S = Q K^T are
// accumulated in tensor memory; the thread that owns a row reads its 128 scores, keeps the row's maximum and sum, and writes
// the probabilities back over the scores as 16-bit lanes, which are the A operand of O += P V there.  V lies in shared memory
// as the cache has it (keys by lanes) and is taken as an MN-major operand, so nothing is transposed.
//
//   warps 0-3, 4-7   the rows of the first and of the second tile, a thread each
//   warp 8           one thread issues the products
//   warp 9           brings keys and values through TMA, a box per page (or per 128 rows of a larger one)
//
// The two tiles take turns: while one's scores become probabilities, the other's products run.  A tile's next scores follow
// its own probabilities' product, since both use its columns of tensor memory, so per pair of tiles the chain is two products
// and one softmax for each.  The output is only rescaled when a row's maximum has grown by more than 2^8 (it is exact
// arithmetic up to rounding whichever maximum is used; the sums stay in f32 and the 16-bit probabilities below 2^8), which
// after the first tiles is rare.  Every wait is bounded.
#include <algorithm>
#include <mutex>

#include "decoder_device.cuh"
#include "umma_kernel.cuh"

namespace oxb {
namespace k {

namespace umma {

constexpr int PR_KEYS = 128, PR_ROWS = 128;
constexpr int PR_THREADS = 384;  // three warpgroups; the last two warps of the third idle
constexpr float PR_GROWTH = 8.f;  // log2 of how far probabilities may exceed 1 before the output is rescaled

template <int KD>
struct PromptShape {
  static constexpr int kHalves = KD / 64;                 // 128-byte wide pieces of a head
  static constexpr uint32_t kTile = kHalves * 16384u;     // 128 rows
  static constexpr int kStages = KD == 64 ? 8 : 5;        // tiles of keys and of values in flight
  static constexpr uint32_t kSmem = (2 + kStages) * kTile + 1024u;
  static constexpr uint32_t kScores = 0, kOut = 256;      // columns of tensor memory: two tiles of each
};

struct alignas(64) PromptParams {
  CUtensorMap keys, values;
  PagedAttention a;
  int box, least_rows;
  uint32_t idesc_s, idesc_o;
  float slope;
  uint32_t flip;
  int mute;
};

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, int c2, int c3) {
  asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
               "l"((uint64_t)map), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
               : "memory");
}
// A from tensor memory (16-bit lanes, two to a column), B from shared memory
__device__ __forceinline__ void tc_mma_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t db, uint32_t idesc, uint32_t accumulate) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(tmem_d), "r"(tmem_a), "l"(db), "r"(idesc),
               "r"(accumulate)
               : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]),
               "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
               : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
      "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_pair(float lo, float hi, __half*) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *(const uint32_t*)&h;
}
__device__ __forceinline__ uint32_t pack_pair(float lo, float hi, __nv_bfloat16*) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *(const uint32_t*)&h;
}

template <typename T, int KD>
__global__ void __launch_bounds__(PR_THREADS, 1) umma_prompt_kernel(const __grid_constant__ PromptParams p) {
  using S = PromptShape<KD>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t bar_q, bar_full[S::kStages], bar_empty[S::kStages], bar_scores[2], bar_probs[2], bar_out[2], bar_tail;
  __shared__ uint32_t tmem_base_slot;
  __shared__ int abort_flag;
  const PagedAttention& a = p.a;
  const int warp = (int)(threadIdx.x >> 5), lane = (int)(threadIdx.x & 31), group = a.heads / a.kv_heads;
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* const base_ptr = smem_raw + (base - smem_u32(smem_raw));
  volatile int* const abortp = &abort_flag;
  pdl_enter();

  // ---- this block's sequence, rows and key head: every warp looks for itself ----
  int b = -1, kv = 0, row0 = 0;
  Sequence q{0, 0, 0};
  bool bad = false;
  {
    long long left = blockIdx.x;
    for (int first = 0; first < a.t.sequences; first += 32) {
      Sequence s{0, 0, 0};
      bool wrong = false;
      if (first + lane < a.t.sequences) s = sequence_of(a.t, first + lane, &wrong);
      const long long rows = (long long)s.rows * group;
      const int blocks = rows >= p.least_rows ? (int)((rows + 2 * PR_ROWS - 1) / (2 * PR_ROWS)) : 0;
      const int items = blocks * a.kv_heads;
      int sum = items;
#pragma unroll
      for (int o = 1; o < 32; o *= 2) {
        const int up = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += up;
      }
      const int all = __shfl_sync(0xffffffffu, sum, 31);
      if (left >= all) {
        left -= all;
        continue;
      }
      const int who = __ffs(__ballot_sync(0xffffffffu, sum > left)) - 1;
      const int item = (int)left - __shfl_sync(0xffffffffu, sum - items, who);
      b = first + who;
      q.first = __shfl_sync(0xffffffffu, s.first, who), q.rows = __shfl_sync(0xffffffffu, s.rows, who), q.length = __shfl_sync(0xffffffffu, s.length, who);
      bad = __shfl_sync(0xffffffffu, wrong ? 1 : 0, who) != 0;
      kv = item % a.kv_heads;
      row0 = (__shfl_sync(0xffffffffu, blocks, who) - 1 - item / a.kv_heads) * 2 * PR_ROWS;  // the rows with the most keys first
      break;
    }
  }
  if (b < 0) return;
  if (bad && threadIdx.x == 0) report(a.err, kErrLengths);
  const int rows = q.rows * group;
  // keys that the last row of tile t sees, in tiles
  auto tiles_of = [&](int t) {
    const int last = min(rows, row0 + (t + 1) * PR_ROWS) - 1;
    if (row0 + t * PR_ROWS >= rows) return 0;
    return (max(0, q.length - q.rows + last / group + 1) + PR_KEYS - 1) / PR_KEYS;
  };
  const int nt[2] = {tiles_of(0), tiles_of(1)}, most = max(nt[0], nt[1]);

  if (threadIdx.x == 0) {
    abort_flag = 0;
    mbar_init(smem_u32(&bar_q), 8);
    for (int i = 0; i < S::kStages; ++i) mbar_init(smem_u32(&bar_full[i]), 1), mbar_init(smem_u32(&bar_empty[i]), 1);
    for (int t = 0; t < 2; ++t) mbar_init(smem_u32(&bar_scores[t]), 1), mbar_init(smem_u32(&bar_probs[t]), 4), mbar_init(smem_u32(&bar_out[t]), 1);
    mbar_init(smem_u32(&bar_tail), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 8) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base_slot)), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_base_slot;
  auto give_up = [&](int code) {
    if (!*abortp) {
      *abortp = 1;
      atomicExch(a.err, code);
    }
  };
  const uint32_t q_off = 0, ring = base + 2 * S::kTile;
  // rows of the last tile of values that lie behind the sequence but in a page that was brought
  const int tail0 = q.length % p.box == 0 ? 0 : q.length - (most - 1) * PR_KEYS, tail1 = (tail0 + p.box - 1) / p.box * p.box;
  const bool tail = most > 0 && most * PR_KEYS > q.length && q.length % p.box != 0;

  // 168 registers a thread at the launch, 64512 together: 216 for the rows' warpgroups and 72 for the third are 64512 again
  if (warp >= 8) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
  if (warp == 9) {
    // ---------------- keys and values ----------------
    const int boxes = PR_KEYS / p.box;
    const int* const table = a.t.page_table + (int64_t)b * a.t.max_pages;
    auto page_of = [&](int j) -> int {  // of this lane's box of tile j; behind the sequence, and in place of what is no page: the zeros behind the cache
      const int key = j * PR_KEYS + lane * p.box;
      if (lane >= boxes || j >= most || key >= q.length) return (int)a.t.pages;
      const int page = table[key / a.t.page];
      if (page >= 0 && page < a.t.pages) return page;
      if (!bad) report(a.err, kErrPage);
      return (int)a.t.pages;
    };
    int page = page_of(0);
    bool ok = true;
    for (int j = 0; j < most && ok; ++j) {
      const int next = page_of(j + 1);
#pragma unroll 1
      for (int kind = 0; kind < 2 && ok; ++kind) {
        const int n = 2 * j + kind, stage = n % S::kStages;
        if (n >= S::kStages) ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&bar_empty[stage]), ((n / S::kStages) & 1u) ^ 1u, abortp));
        if (!ok) {
          if (lane == 0) give_up(41);
          break;
        }
        const uint32_t bar = smem_u32(&bar_full[stage]), dst = ring + stage * S::kTile;
        if (lane == 0) mbar_expect_tx(bar, S::kTile);
        __syncwarp();
        if (lane < boxes)
#pragma unroll
          for (int h = 0; h < S::kHalves; ++h)
            tma_load_4d(dst + h * 16384u + lane * p.box * 128u, kind == 0 ? &p.keys : &p.values, bar, h * 64, kv, (j * PR_KEYS + lane * p.box) % a.t.page, page);
      }
      page = next;
    }
    if (ok && tail) {  // what a page holds behind the sequence may be anything, and 0 times it is not always 0
      const int n = 2 * most - 1, stage = n % S::kStages;
      ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&bar_full[stage]), (n / S::kStages) & 1u, abortp));
      if (ok) {
        uint8_t* const v = base_ptr + 2 * S::kTile + stage * S::kTile;
        for (int i = lane; i < (tail1 - tail0) * 8 * S::kHalves; i += 32) {
          const int r = tail0 + i / (8 * S::kHalves), c = i % (8 * S::kHalves);
          *(uint4*)(v + (c / 8) * 16384 + r * 128 + (c % 8) * 16) = make_uint4(0, 0, 0, 0);  // all of the row: the swizzle does not matter
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&bar_tail));
      } else if (lane == 0) {
        give_up(42);
      }
    }
  } else if (warp == 8) {
    // ---------------- products ----------------
    if (elect_one() && most > 0) {
      auto wait = [&](uint64_t& bar, uint32_t parity, int code) {
        if (mbar_wait(smem_u32(&bar), parity, abortp)) return true;
        give_up(code);
        return false;
      };
      const uint64_t kmajor = make_smem_desc(0, 128);
      // values: 64 lanes by 8 keys to a swizzle atom of 1024 bytes, atoms of the next 8 keys 1024 and of the next 64 lanes 16384 behind
      const uint64_t vmajor = ((uint64_t)(16384u >> 4) << 16) | ((uint64_t)(1024u >> 4) << 32) | (1ull << 46) | (2ull << 61);
      auto full = [&](int n) { return wait(bar_full[n % S::kStages], (n / S::kStages) & 1u, 43); };
      auto scores = [&](int t, int n) {  // S_t = Q_t K^T with the keys of slot n
        const uint32_t qa = base + q_off + t * S::kTile, ka = ring + (n % S::kStages) * S::kTile;
#pragma unroll
        for (int k = 0; k < KD / 16; ++k) {
          const uint32_t off = (uint32_t)(k / 4) * 16384u + (uint32_t)(k % 4) * 32u;
          tc_mma_one<KIND_F16>(tmem + S::kScores + t * 128, kmajor | (((qa + off) >> 4) & 0x3fffu), kmajor | (((ka + off) >> 4) & 0x3fffu), p.idesc_s, k > 0 ? 1u : 0u);
        }
        tc_commit<false>(smem_u32(&bar_scores[t]));
      };
      bool ok = wait(bar_q, 0u, 44) && full(0);
      if (ok) {
        tc_fence_after();
        for (int t = 0; t < 2; ++t)
          if (nt[t] > 0) scores(t, 0);
        tc_commit<false>(smem_u32(&bar_empty[0]));
      }
      for (int j = 0; j < most && ok; ++j) {
        ok = full(2 * j + 1) && (j + 1 >= most || full(2 * j + 2));
        if (ok && tail && j == most - 1) ok = wait(bar_tail, 0u, 45);
        for (int t = 0; t < 2 && ok; ++t) {
          if (j >= nt[t]) continue;
          ok = wait(bar_probs[t], j & 1u, 46);
          if (!ok) break;
          tc_fence_after();
          const uint32_t va = ring + ((2 * j + 1) % S::kStages) * S::kTile;
#pragma unroll
          for (int k = 0; k < PR_KEYS / 16; ++k)
            tc_mma_ts(tmem + S::kOut + t * KD, tmem + S::kScores + t * 128 + k * 8, vmajor | (((va + k * 2048u) >> 4) & 0x3fffu), p.idesc_o, j + k > 0 ? 1u : 0u);
          if (j + 1 < nt[t]) scores(t, 2 * j + 2);
          else tc_commit<false>(smem_u32(&bar_out[t]));
        }
        if (!ok) break;
        tc_commit<false>(smem_u32(&bar_empty[(2 * j + 1) % S::kStages]));
        if (j + 1 < most) tc_commit<false>(smem_u32(&bar_empty[(2 * j + 2) % S::kStages]));
      }
    }
    __syncwarp();
  }
  } else {
    // ---------------- rows ----------------
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    const int t = warp >> 2, quarter = warp & 3, first_row = row0 + t * PR_ROWS;
    {  // the tile's queries, as TMA would have laid them out: 16 bytes c of a row lie at c ^ (row & 7)
      uint8_t* const dst = base_ptr + q_off + t * S::kTile;
      constexpr int CH = KD / 8;
      for (int i = (int)threadIdx.x & 127; i < PR_ROWS * CH; i += 128) {
        const int r = i / CH, c = i % CH, row = first_row + r;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (row < rows && c * 8 < a.size && !p.mute) {
          v = *(const uint4*)((const T*)a.q + ((int64_t)(q.first + row / group) * a.heads + kv * group + row % group) * a.size + c * 8);
          v.x ^= p.flip, v.y ^= p.flip, v.z ^= p.flip, v.w ^= p.flip;
        }
        *(uint4*)(dst + (c / 8) * 16384 + r * 128 + (((c % 8) ^ (r & 7)) << 4)) = v;
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&bar_q));
    }
    const int row = first_row + quarter * 32 + lane;
    const int limit = row < rows ? max(0, q.length - q.rows + row / group + 1) : 0;
    const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
    const uint32_t s_col = tmem + lane_base + S::kScores + t * 128, o_col = tmem + lane_base + S::kOut + t * KD;
    const uint64_t slope2 = both(p.slope);
    float top = -INFINITY, sum = 0.f;  // the maximum that the output is relative to, and the sum
    bool whole = true;
    for (int j = 0; j < nt[t]; ++j) {
      if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&bar_scores[t]), j & 1u, abortp))) {
        if (lane == 0) give_up(47);
        whole = false;
        break;
      }
      tc_fence_after();
      uint32_t r[4][32];
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_ld32_nowait(s_col + 32 * c, r[c]);
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_ld_wait_for(r[c]);
      const int seen = limit - j * PR_KEYS;
      if (__any_sync(0xffffffffu, seen < PR_KEYS)) {
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (c * 32 + i >= seen) r[c][i] = 0xff800000u;
      }
      float mx[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        mx[c] = __uint_as_float(r[c][0]);
#pragma unroll
        for (int i = 1; i < 32; ++i) mx[c] = fmaxf(mx[c], __uint_as_float(r[c][i]));
      }
      const float high = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
      if (j == 0) {
        top = high;
      } else if (__any_sync(0xffffffffu, (high - top) * p.slope > PR_GROWTH)) {
        // these scores are complete, so is the product before them: the output may be rewritten
        const float next = fmaxf(top, high);
        const float keep = top == -INFINITY ? 0.f : ex2((top - next) * p.slope);
        top = next;
        sum *= keep;
#pragma unroll
        for (int c = 0; c < KD / 32; ++c) {
          uint32_t o[32];
          tmem_ld32_nowait(o_col + 32 * c, o);
          tmem_ld_wait_for(o);
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * keep);
          tmem_st32(o_col + 32 * c, o);
        }
      }
      const float bias = top == -INFINITY ? 0.f : top * p.slope;
      uint64_t part = 0;  // two sums
      const uint64_t bias2 = both(-bias);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t w[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          float x, y;
          unpack2(fmap(pack2(__uint_as_float(r[c][2 * i]), __uint_as_float(r[c][2 * i + 1])), slope2, bias2), x, y);
          x = ex2(x), y = ex2(y);
          part = addp(part, pack2(x, y));
          w[i] = pack_pair(x, y, (T*)nullptr);
        }
        tmem_st16(s_col + 16 * c, w);
      }
      float even, odd;
      unpack2(part, even, odd);
      sum += even + odd;
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&bar_probs[t]));
    }
    if (whole) {
      const bool some = nt[t] > 0;
      if (some && !__all_sync(0xffffffffu, mbar_wait(smem_u32(&bar_out[t]), 0u, abortp))) {
        if (lane == 0) give_up(48);
      } else {
        tc_fence_after();
        const float inv = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;  // NaN where a key was
        T* const out = (T*)a.out + ((int64_t)(q.first + (row < rows ? row / group : 0)) * a.heads + kv * group + row % group) * a.size;
#pragma unroll
        for (int c = 0; c < KD / 32; ++c) {
          uint32_t o[32];
          if (some) {
            tmem_ld32_nowait(o_col + 32 * c, o);
            tmem_ld_wait_for(o);
          }
          if (row < rows)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (c * 32 + e * 8 < a.size) {
                uint32_t w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i)
                  w[i] = some && limit > 0 ? pack_pair(__uint_as_float(o[e * 8 + 2 * i]) * inv, __uint_as_float(o[e * 8 + 2 * i + 1]) * inv, (T*)nullptr) : 0u;
                *(uint4*)(out + c * 32 + e * 8) = make_uint4(w[0], w[1], w[2], w[3]);
              }
        }
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
  if (warp == 8) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base_slot), "r"(512) : "memory");
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

// Boxes of 64 lanes by `box` rows of one head of one page; lanes behind the head and pages behind the cache read as zeros.
void encode_cache(CUtensorMap* map, const PagedAttention& a, const void* cache, int box) {
  const cuuint64_t row = (cuuint64_t)a.kv_heads * a.size * 2;
  cuuint64_t dims[4] = {(cuuint64_t)a.size, (cuuint64_t)a.kv_heads, (cuuint64_t)a.t.page, (cuuint64_t)a.t.pages};
  cuuint64_t strides[3] = {(cuuint64_t)a.size * 2, row, row * a.t.page};
  cuuint32_t boxes[4] = {64, 1, (cuuint32_t)box, 1}, steps[4] = {1, 1, 1, 1};
  EncodeTiledFn encode = tiled_encoder();
  if (!encode || encode(map, a.dt == DT::F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(cache), dims, strides, boxes, steps,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
    OXB_FAIL("OxiPagedAttention: the driver refused a tensor map of the cache");
}

template <typename T, int KD>
void launch_prompt(const PagedAttention& a, int least_rows, cudaStream_t s) {
  using S = PromptShape<KD>;
  static std::mutex mu;
  static bool have[64] = {};
  int device = 0;
  OXB_CUDA(cudaGetDevice(&device));
  {
    std::lock_guard<std::mutex> lock(mu);
    if (device < 0 || device >= 64 || !have[device]) {
      OXB_CUDA(cudaFuncSetAttribute(umma_prompt_kernel<T, KD>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)S::kSmem));
      if (device >= 0 && device < 64) have[device] = true;
    }
  }
  PromptParams p{};
  p.a = a;
  p.box = std::min(a.t.page & -a.t.page, PR_KEYS);  // the largest power of two that divides a page
  p.least_rows = least_rows;
  encode_cache(&p.keys, a, a.key_cache, p.box);
  encode_cache(&p.values, a, a.value_cache, p.box);
  // kind::f16: f32 accumulator, A and B in the cache's type; scores: both K-major, 128 x 128; output: B MN-major, 128 x KD
  const uint32_t type = a.dt == DT::F16 ? 0u : 1u, common = (1u << 4) | (type << 7) | (type << 10) | ((128u >> 4) << 24);
  p.idesc_s = common | ((128u >> 3) << 17);
  p.idesc_o = common | (1u << 16) | (((uint32_t)KD >> 3) << 17);
  p.slope = (a.scale == 0.f ? 1.f : std::fabs(a.scale)) * 1.4426950408889634f;
  p.flip = a.scale < 0.f ? 0x80008000u : 0u;
  p.mute = a.scale == 0.f;
  // no more blocks than these: a sequence of r packed rows has at most r / 256 + 1, and r is at least least_rows
  const int64_t rows = a.t.tokens * (a.heads / a.kv_heads), blocks = a.kv_heads * (rows / (2 * PR_ROWS) + std::min<int64_t>(a.t.sequences, rows / least_rows));
  if (blocks > 0) launch(umma_prompt_kernel<T, KD>, dim3((unsigned)blocks), dim3(PR_THREADS), S::kSmem, s, p);
}

}  // namespace

void paged_attention_prompts(const PagedAttention& a, int least_rows, cudaStream_t s) {
  if (a.dt == DT::F16) a.size <= 64 ? launch_prompt<__half, 64>(a, least_rows, s) : launch_prompt<__half, 128>(a, least_rows, s);
  else a.size <= 64 ? launch_prompt<__nv_bfloat16, 64>(a, least_rows, s) : launch_prompt<__nv_bfloat16, 128>(a, least_rows, s);
}

}  // namespace k
}  // namespace oxb
