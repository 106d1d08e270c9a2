// Causal attention of many packed rows over the pages of a cache, on tcgen05: scores and output never leave the SM.
//
// A work item is two tiles of at most 128 packed rows (whole tokens) of one key head; its keys are walked 128 at a time.
// Scores S = Q K^T are accumulated in tensor memory; the thread that owns a row reads its 128 scores, keeps the row's maximum
// and sum, and writes the probabilities back over the scores as 16-bit lanes, which are the A operand of O += P V there.  V
// lies in shared memory as the cache has it (keys by lanes) and is taken as an MN-major operand, so nothing is transposed.
//
//   warps 0-3, 4-7   the rows of the first and of the second tile, a thread each
//   warp 8           one thread issues the products
//   warp 9           brings queries, keys and values through TMA, a box per page (or per 128 rows of a larger one)
//   warp 10          finds the block's items, two ahead
//
// The two tiles take turns: while one's scores become probabilities, the other's products run.  A tile's next scores follow
// its own probabilities' product, since both use its columns of tensor memory.  The output is only rescaled when a row's
// maximum has grown by more than 2^8 (f16: 2^4; it is exact arithmetic up to rounding whichever maximum is used; the sums stay in
// f32 and the 16-bit probabilities below 2^8, f16's below 2^15), which after the first tiles is rare.
//
// One block per SM takes an equal run of all items' key tiles (PromptWork), so that one long prompt, many short ones and a few
// rows behind a long past fill the chip alike; items run into one another without a pause: the next item's queries are brought
// when the last scores of this one are done, and its first scores run while this one's output leaves.  An item that a border
// between blocks cuts leaves its parts in the workspace, and whoever brings the last part joins them in the order of the keys.
// Every wait is bounded.
//
// A step (both tiles by 128 keys of 128 lanes) takes 4000 cycles, of which the products are 2048 and the exponentials as many:
// 8192 tokens of 32 heads on 8 take 557 us, 987 TFLOP/s, at the power cap.  64 keys a step in two buffers (products of 64
// columns run at half rate), polynomials for a part of the exponentials and a second issuing thread were no faster.
#include <algorithm>
#include <mutex>

#include "decoder_device.cuh"
#include "decoder_schedule.hpp"
#include "umma_kernel.cuh"

namespace oxb {
namespace k {

namespace umma {

constexpr int PR_KEYS = 128, PR_ROWS = 128;
constexpr int PR_THREADS = 384;  // three warpgroups; the last two warps of the third idle
constexpr int PR_LEAST_STEPS = 6;  // steps that a block takes at least: below, joining the parts costs more than the keys
constexpr float PR_FAR = 1024.f;  // product of maximum and slope above which the maximum is taken off first (kFar of paged_attention.cu)
// log2 of what the probability of the maximum is written as (kLift of paged_attention.cu), and of how far others may exceed it before
// the output is rescaled: together below f16's 2^16.
template <typename T>
constexpr float PR_LIFT = 0.f;
template <>
constexpr float PR_LIFT<__half> = 11.f;
template <typename T>
constexpr float PR_GROWTH = 8.f;
template <>
constexpr float PR_GROWTH<__half> = 4.f;

template <int KD>
struct PromptShape {
  static constexpr int kHalves = KD / 64;                 // 128-byte wide pieces of a head
  static constexpr uint32_t kTile = kHalves * 16384u;     // 128 rows
  static constexpr int kStages = KD == 64 ? 8 : 5;        // tiles of keys and of values in flight
  static constexpr uint32_t kSmem = (2 + kStages) * kTile + 1024u;
  static constexpr uint32_t kScores = 0, kOut = 256;      // columns of tensor memory: two tiles of each
};

// What a part of an item leaves in the workspace, two to a block ([0] of an item that began in an earlier block, [1] of one
// that goes on in the next): the output as [KD / 4][256 rows] float4, then maximum and sum of each row.
template <int KD>
constexpr size_t kPromptPart = (size_t)2 * PR_ROWS * (KD + 2);

struct alignas(64) PromptParams {
  CUtensorMap queries, keys, values;
  PagedAttention a;
  float* parts;
  int* counters;  // two to a block
  int box, least_rows, span;
  uint32_t idesc_s, idesc_o;
  float slope;
  uint32_t flip;
  int mute;
};

// A part of an item, as the finder hands it to the other warps.
struct PromptItem {
  int valid, b, bad;
  int first, rows, length;  // of the sequence
  int token0, kv;           // first new token of the item's first tile, key head
  int j0, j1, tiles[2];     // key tiles of the part; of the whole item for each tile of rows
  int c0, c1[2];            // blocks that hold the item's first key tile and the last one of each tile of rows
};

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, int c2, int c3) {
  asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
               "l"((uint64_t)map), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
               : "memory");
}
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, int c2) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst), "l"((uint64_t)map), "r"(bar), "r"(c0),
               "r"(c1), "r"(c2)
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
// with its wait
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\ttcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// in 32 bits where both fit, as they do for all but absurd sizes: the division of 64-bit numbers is a hundred instructions
__device__ __forceinline__ long long quotient(long long x, long long y) {
  return ((unsigned long long)(x | y) >> 32) ? x / y : (long long)((unsigned)x / (unsigned)y);
}
// The largest of three; NaN where one is.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float y;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}
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
  __shared__ __align__(8) uint64_t bar_item_full[2], bar_item_empty[2], bar_q_full, bar_q_empty, bar_full[S::kStages], bar_empty[S::kStages], bar_scores[2], bar_probs[2], bar_out[2], bar_tail;
  __shared__ PromptItem items[2];
  __shared__ long long scan[PR_THREADS / 32], start_before;
  __shared__ int start_b, last_part[2];
  __shared__ uint32_t tmem_base_slot;
  __shared__ int abort_flag;
  const PagedAttention& a = p.a;
  const int warp = (int)(threadIdx.x >> 5), lane = (int)(threadIdx.x & 31), group = a.heads / a.kv_heads;
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* const base_ptr = smem_raw + (base - smem_u32(smem_raw));
  volatile int* const abortp = &abort_flag;
  if (threadIdx.x == 0) {
    abort_flag = 0;
    start_b = -1;
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&bar_item_full[i]), 1), mbar_init(smem_u32(&bar_item_empty[i]), 10);  // read by the loader, the issuer and eight warps of rows
      mbar_init(smem_u32(&bar_scores[i]), 1), mbar_init(smem_u32(&bar_probs[i]), 4), mbar_init(smem_u32(&bar_out[i]), 1);
    }
    mbar_init(smem_u32(&bar_q_full), 1), mbar_init(smem_u32(&bar_q_empty), 1), mbar_init(smem_u32(&bar_tail), 1);
    for (int i = 0; i < S::kStages; ++i) mbar_init(smem_u32(&bar_full[i]), 1), mbar_init(smem_u32(&bar_empty[i]), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  // The successor is let in only behind the allocation below: a block of it that fits beside this one and takes its columns of
  // tensor memory first would hold them until this grid ends, which this block's allocation would then never let it.
  asm volatile("griddepcontrol.wait;" ::: "memory");

  // ---- all sequences' steps, and the sequence that this block's first step lies in ----
  auto work_of = [&](const Sequence& s) {
    return PromptWork{(long long)s.rows * group >= p.least_rows ? s.rows : 0, s.length - s.rows, p.span, a.kv_heads};
  };
  long long total = 0, per = 0, begin = 0;
  {
    // Up to PR_THREADS sequences a thread has its own in hand when the sum of all is known; beyond, they are gone through twice.
    const int rounds = (a.t.sequences + PR_THREADS - 1) / PR_THREADS;
    for (int pass = 0; pass < (rounds > 1 ? 2 : 1); ++pass) {
      long long seen = 0;
      for (int round = 0; round < rounds; ++round) {
        const int b = round * PR_THREADS + (int)threadIdx.x;
        long long mine = 0, sum;
        if (b < a.t.sequences) {
          bool bad;
          mine = work_of(sequence_of(a.t, b, &bad)).total();
        }
        sum = mine;
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
          const long long up = __shfl_up_sync(0xffffffffu, sum, o);
          if (lane >= o) sum += up;
        }
        if (lane == 31) scan[warp] = sum;
        __syncthreads();
        sum += seen;
        for (int w = 0; w < PR_THREADS / 32; ++w) {
          if (w < warp) sum += scan[w];
          seen += scan[w];
        }
        if (pass == 0 && round + 1 == rounds) {
          total = seen;
          per = max((long long)PR_LEAST_STEPS, quotient(total + gridDim.x - 1, gridDim.x));
          begin = blockIdx.x * per;
        }
        if ((pass == 1 || rounds == 1) && begin >= sum - mine && begin < sum) start_b = b, start_before = sum - mine;
        __syncthreads();
      }
    }
  }
  const long long stop = min(total, begin + per);
  if (begin >= stop) return;

  if (warp == 8) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base_slot)), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const uint32_t tmem = tmem_base_slot;
  auto give_up = [&](int code) {
    if (!*abortp) {
      *abortp = 1;
      atomicExch(a.err, code);
    }
  };
  const uint32_t ring = base + 2 * S::kTile;
  // item number i of this block, once it is found (each lane asks; false when a wait ran out)
  auto item_ready = [&](uint32_t i) { return mbar_wait(smem_u32(&bar_item_full[i & 1u]), (i >> 1) & 1u, abortp); };
  // Rows [tail0, tail1) of the part's last tile of values lie behind the sequence in a page that was brought.
  auto tail_of = [&](const PromptItem& w, int* tail0, int* tail1) {
    const int end = w.j1 * PR_KEYS;
    if (end <= w.length || w.length % p.box == 0 || w.length <= (w.j1 - 1) * PR_KEYS) return false;
    *tail0 = w.length - (w.j1 - 1) * PR_KEYS;
    *tail1 = (*tail0 + p.box - 1) / p.box * p.box;
    return true;
  };

  if (warp >= 8) {
    // 168 registers a thread at the launch, 64512 together: 216 for the rows' warpgroups and 72 for this one are 64512 again
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    if (warp == 10) {
      // ---------------- items ----------------
      int b = start_b;
      long long at = begin, seq_before = start_before;
      uint32_t i = 0;
      bool ok = true;
      Sequence q{0, 0, 0};
      bool bad = false;
      PromptWork w{0, 0, p.span, a.kv_heads};
      int block = -1, kv = 0;
      long long item_at = 0;  // the item's first step
      while (ok) {
        PromptItem it{};
        while (at < stop && !it.valid) {
          if (block < 0) {  // the first item of a sequence (or of this block)
            q = sequence_of(a.t, b, &bad);
            w = work_of(q);
            // (a search by before() took 10 us of divisions)
            long long inside = at - seq_before;
            block = w.block_of(&inside, [&](auto steps, long long inside) {
              const long long mine = steps(lane);
              long long sum = mine;
#pragma unroll
              for (int o = 1; o < 32; o *= 2) {
                const long long up = __shfl_up_sync(0xffffffffu, sum, o);
                if (lane >= o) sum += up;
              }
              const unsigned in = __ballot_sync(0xffffffffu, sum > inside);
              const int who = in ? __ffs(in) - 1 : 31;
              return PromptWork::Found{in ? who : 32, __shfl_sync(0xffffffffu, in ? sum - mine : sum, who)};
            });
            const int steps = w.steps(block);
            kv = (int)quotient(inside, steps);
            item_at = at - (inside - (long long)kv * steps);
          }
          const long long item_end = item_at + w.steps(block), end = min(stop, item_end);
          it.j0 = (int)max(0LL, at - item_at - PromptWork::kBegin), it.j1 = (int)(end - item_at - PromptWork::kBegin);
          if (it.j1 > it.j0) {
            it.valid = 1, it.b = b, it.bad = bad ? 1 : 0;
            it.first = q.first, it.rows = q.rows, it.length = q.length;
            it.token0 = block * 2 * p.span, it.kv = kv;
            it.c0 = (int)quotient(item_at + PromptWork::kBegin, per);
            for (int t = 0; t < 2; ++t) {
              it.tiles[t] = w.tiles_of(block, t);
              it.c1[t] = (int)quotient(item_at + PromptWork::kBegin + max(it.tiles[t], 1) - 1, per);
            }
          }
          at = end;
          if (end == item_end) {  // on to the next item
            item_at = item_end;
            if (++kv == a.kv_heads) {
              kv = 0;
              if (++block == w.blocks()) {
                seq_before += w.total();
                block = -1;
                int next = -1;
                for (int first = b + 1; first < a.t.sequences && next < 0; first += 32) {
                  bool wrong;
                  const bool has = first + lane < a.t.sequences && work_of(sequence_of(a.t, first + lane, &wrong)).rows > 0;
                  const unsigned any = __ballot_sync(0xffffffffu, has);
                  if (any) next = first + __ffs(any) - 1;
                }
                if (next < 0) at = stop;
                b = next;
              }
            }
          }
        }
        const uint32_t slot = i & 1u;
        if (i >= 2 && !__all_sync(0xffffffffu, mbar_wait(smem_u32(&bar_item_empty[slot]), ((i >> 1) & 1u) ^ 1u, abortp))) {
          if (lane == 0) give_up(49);
          ok = false;
          break;
        }
        if (lane == 0) {
          items[slot] = it;
          if (it.valid && it.bad) report(a.err, kErrLengths);
          mbar_arrive(smem_u32(&bar_item_full[slot]));
        }
        ++i;
        if (!it.valid) break;
      }
    } else if (warp == 9) {
      // ---------------- queries, keys and values ----------------
      const int boxes = PR_KEYS / p.box, box = lane % boxes, half = lane / boxes;  // a lane for each box of 64 lanes
      int n = 0;  // tiles brought so far
      uint32_t tails = 0;
      bool ok = true;
      for (uint32_t i = 0; ok; ++i) {
        if (!__all_sync(0xffffffffu, item_ready(i))) {
          if (lane == 0) give_up(40);
          break;
        }
        const PromptItem w = items[i & 1u];
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&bar_item_empty[i & 1u]));
        if (!w.valid) break;
        const int* const table = a.t.page_table + (int64_t)w.b * a.t.max_pages;
        auto page_of = [&](int j) -> int {  // of this lane's box of tile j; behind the sequence, and in place of what is no page: the zeros behind the cache
          const int key = j * PR_KEYS + box * p.box;
          if (half >= S::kHalves || j >= w.j1 || key >= w.length) return (int)a.t.pages;
          const int page = table[key / a.t.page];
          if (page >= 0 && page < a.t.pages) return page;
          if (!w.bad) report(a.err, kErrPage);
          return (int)a.t.pages;
        };
        int page = page_of(w.j0);
        if (i > 0) ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&bar_q_empty), (i - 1u) & 1u, abortp));
        if (!ok) {
          if (lane == 0) give_up(50);
          break;
        }
        if (lane == 0) {
          mbar_expect_tx(smem_u32(&bar_q_full), 2u * S::kHalves * 128u * (uint32_t)(group * p.span));
          for (int t = 0; t < 2; ++t)
            for (int h = 0; h < S::kHalves; ++h)
              tma_load_3d(base + t * S::kTile + h * 16384u, &p.queries, smem_u32(&bar_q_full), h * 64, w.kv * group, w.first + w.token0 + t * p.span);
        }
        __syncwarp();
        for (int j = w.j0; j < w.j1 && ok; ++j) {
          const int next = page_of(j + 1);
#pragma unroll 1
          for (int kind = 0; kind < 2; ++kind, ++n) {
            const int stage = n % S::kStages;
            if (n >= S::kStages) ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&bar_empty[stage]), ((n / S::kStages) & 1u) ^ 1u, abortp));
            if (!ok) {
              if (lane == 0) give_up(41);
              break;
            }
            const uint32_t bar = smem_u32(&bar_full[stage]), dst = ring + stage * S::kTile;
            if (lane == 0) mbar_expect_tx(bar, S::kTile);
            __syncwarp();
            if (lane < boxes * S::kHalves)
              tma_load_4d(dst + half * 16384u + box * p.box * 128u, kind == 0 ? &p.keys : &p.values, bar, half * 64, w.kv, (j * PR_KEYS + box * p.box) % a.t.page, page);
          }
          page = next;
        }
        int tail0, tail1;
        if (ok && tail_of(w, &tail0, &tail1)) {  // what a page holds behind the sequence may be anything, and 0 times it is not always 0
          const int stage = (n - 1) % S::kStages;
          ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&bar_full[stage]), ((n - 1) / S::kStages) & 1u, abortp));
          if (!ok) {
            if (lane == 0) give_up(42);
            break;
          }
          uint8_t* const v = base_ptr + 2 * S::kTile + stage * S::kTile;
          for (int e = lane; e < (tail1 - tail0) * 8 * S::kHalves; e += 32) {
            const int r = tail0 + e / (8 * S::kHalves), c = e % (8 * S::kHalves);
            *(uint4*)(v + (c / 8) * 16384 + r * 128 + (c % 8) * 16) = make_uint4(0, 0, 0, 0);  // all of the row: the swizzle does not matter
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&bar_tail));
          ++tails;
        }
      }
    } else if (warp == 8) {
      // ---------------- products ----------------
      if (elect_one()) {
        auto wait = [&](uint64_t& bar, uint32_t parity, int code) {
          if (mbar_wait(smem_u32(&bar), parity, abortp)) return true;
          give_up(code);
          return false;
        };
        // Whole descriptors, so that an instruction costs one addition.  One thread for both tiles of rows: their products follow
        // one another whole, and the first is done early.  A thread for each (2048 tokens 65 -> 73 us) had them share the pipe.
        const uint64_t queries = make_smem_desc(base, 128), keys = make_smem_desc(ring, 128);
        // values: 64 lanes by 8 keys to a swizzle atom of 1024 bytes, atoms of the next 8 keys 1024 and of the next 64 lanes 16384 behind
        const uint64_t values = ((uint64_t)(16384u >> 4) << 16) | ((uint64_t)(1024u >> 4) << 32) | (1ull << 46) | (2ull << 61) | (ring >> 4);
        auto full = [&](int n) { return wait(bar_full[n % S::kStages], (n / S::kStages) & 1u, 43); };
        auto scores = [&](int t, int n) {  // S_t = Q_t K^T with the keys of slot n
          const uint64_t q_at = queries + t * (S::kTile >> 4), k_at = keys + (uint32_t)(n % S::kStages) * (S::kTile >> 4);
          const uint32_t to = tmem + S::kScores + t * 128;
#pragma unroll
          for (int k = 0; k < KD / 16; ++k)
            tc_mma_one<KIND_F16>(to, q_at + (uint32_t)(k / 4) * 1024u + (uint32_t)(k % 4) * 2u, k_at + (uint32_t)(k / 4) * 1024u + (uint32_t)(k % 4) * 2u, p.idesc_s, k > 0 ? 1u : 0u);
          tc_commit<false>(smem_u32(&bar_scores[t]));
        };
        uint32_t probs[2] = {0, 0}, tails = 0;
        int n = 0;
        bool ok = true;
        for (uint32_t i = 0; ok; ++i) {
          if (!item_ready(i)) {
            give_up(44);
            break;
          }
          const PromptItem w = items[i & 1u];
          mbar_arrive(smem_u32(&bar_item_empty[i & 1u]));
          if (!w.valid) break;
          int tail0, tail1;
          const bool tail = tail_of(w, &tail0, &tail1);
          ok = wait(bar_q_full, i & 1u, 44) && full(n);
          if (!ok) break;
          tc_fence_after();
          for (int t = 0; t < 2; ++t)
            if (w.j0 < w.tiles[t]) scores(t, n);
          tc_commit<false>(smem_u32(&bar_empty[n % S::kStages]));
          if (w.j1 - w.j0 == 1) tc_commit<false>(smem_u32(&bar_q_empty));
          for (int j = w.j0; j < w.j1 && ok; ++j, n += 2) {
            const bool more = j + 1 < w.j1;
            ok = full(n + 1) && (!more || full(n + 2));
            if (ok && tail && !more) ok = wait(bar_tail, tails++ & 1u, 45);
            for (int t = 0; t < 2 && ok; ++t) {
              if (j >= w.tiles[t]) continue;
              ok = wait(bar_probs[t], probs[t]++ & 1u, 46);
              if (!ok) break;
              tc_fence_after();
              const uint64_t v_at = values + (uint32_t)((n + 1) % S::kStages) * (S::kTile >> 4);
#pragma unroll
              for (int k = 0; k < PR_KEYS / 16; ++k)
                tc_mma_ts(tmem + S::kOut + t * KD, tmem + S::kScores + t * 128 + k * 8, v_at + k * 128, p.idesc_o, k > 0 ? 1u : (j > w.j0 ? 1u : 0u));
              if (j + 1 < min(w.j1, w.tiles[t])) scores(t, n + 2);
              else tc_commit<false>(smem_u32(&bar_out[t]));
            }
            if (!ok) break;
            tc_commit<false>(smem_u32(&bar_empty[(n + 1) % S::kStages]));
            if (more) tc_commit<false>(smem_u32(&bar_empty[(n + 2) % S::kStages]));
            if (j + 2 == w.j1) tc_commit<false>(smem_u32(&bar_q_empty));
          }
        }
      }
      __syncwarp();
    }
  } else {
    // ---------------- rows ----------------
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    const int t = warp >> 2, quarter = warp & 3, r_tile = quarter * 32 + lane, r_part = t * PR_ROWS + r_tile;
    const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
    const uint32_t s_col = tmem + lane_base + S::kScores + t * 128, o_col = tmem + lane_base + S::kOut + t * KD;
    const uint64_t slope2 = both(p.slope);
    float growth = 0.f, bias = 0.f;  // of a maximum before the output is rescaled (far from 0 none: every step comes by); what is added to scaled scores
    uint32_t done = 0, outs = 0;  // key tiles and parts of this tile of rows so far
    bool whole = true;
    for (uint32_t i = 0; whole; ++i) {
      if (!__all_sync(0xffffffffu, item_ready(i))) {
        if (lane == 0) give_up(40);
        break;
      }
      const volatile PromptItem& w = items[i & 1u];  // read again where it is needed: the loop below has no registers for it
      if (!w.valid) break;
      int limit, j0, j1;
      {
        const int mine = w.token0 + t * p.span + r_tile / group;
        limit = r_tile / group < p.span && mine < w.rows ? max(0, w.length - w.rows + mine + 1) : 0;
        j0 = w.j0, j1 = min(w.j1, w.tiles[t]);
      }
      float top = -INFINITY, sum = 0.f;  // the maximum that the output is relative to, and the sum
#pragma unroll 1
      for (int j = j0; j < j1; ++j, ++done) {
        if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&bar_scores[t]), done & 1u, abortp))) {
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
        if (p.flip | p.mute) {  // a scale of other sign, or of 0
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int e = 0; e < 32; ++e) r[c][e] = p.mute ? 0u : r[c][e] ^ 0x80000000u;
        }
        const int seen = limit - j * PR_KEYS;
        if (__any_sync(0xffffffffu, seen < PR_KEYS)) {
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (c * 32 + e >= seen) r[c][e] = 0xff800000u;
        }
        float mx[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          mx[c] = __uint_as_float(r[c][31]);
#pragma unroll
          for (int e = 0; e < 30; e += 2) mx[c] = max3(mx[c], __uint_as_float(r[c][e]), __uint_as_float(r[c][e + 1]));
          mx[c] = max3(mx[c], __uint_as_float(r[c][30]), mx[c]);
        }
        const float high = max3(max3(mx[0], mx[1], mx[2]), mx[3], mx[3]);
        if (j == j0 || __any_sync(0xffffffffu, !(high <= top + growth))) {
          if (j == j0) {
            top = high;
          } else {
            // these scores are complete, so is the product before them: the output may be rewritten
            const float next = max3(top, high, high);
            const float keep = top == -INFINITY ? 0.f : ex2((top - next) * p.slope);
            top = next;
            sum *= keep;
#pragma unroll 1
            for (int c = 0; c < KD / 16; ++c) {
              uint32_t o[16];
              tmem_ld16(o_col + 16 * c, o);
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * keep);
              tmem_st16(o_col + 16 * c, o);
            }
          }
          bias = top == -INFINITY ? 0.f : fmaf(-top, p.slope, PR_LIFT<T>);
          growth = PR_GROWTH<T> / p.slope;
          // Here, where a step seldom comes: a branch of its own in front of the exponentials cost a long prompt 2.5 %.
          if (__any_sync(0xffffffffu, fabsf(bias) > PR_FAR)) {
            if (top != -INFINITY) {  // scores are -infinity with it
#pragma unroll
              for (int c = 0; c < 4; ++c)
#pragma unroll
                for (int e = 0; e < 32; ++e) r[c][e] = __float_as_uint(__uint_as_float(r[c][e]) - top);
            }
            bias = PR_LIFT<T>, growth = -INFINITY;
          }
        }
        uint64_t part = 0;  // two sums
        const uint64_t bias2 = both(bias);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t out[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            float x, y;
            unpack2(fmap(pack2(__uint_as_float(r[c][2 * e]), __uint_as_float(r[c][2 * e + 1])), slope2, bias2), x, y);
            x = ex2(x), y = ex2(y);
            part = addp(part, pack2(x, y));
            out[e] = pack_pair(x, y, (T*)nullptr);
          }
          tmem_st16(s_col + 16 * c, out);
        }
        float even, odd;
        unpack2(part, even, odd);
        sum += even + odd;
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&bar_probs[t]));
      }
      if (!whole) break;
      const bool some = j0 < j1;
      const int token = r_tile / group, mine = w.token0 + t * p.span + token, c0 = w.c0, c1 = w.c1[t];
      const bool real = token < p.span && mine < w.rows;  // rows behind span * group belong to nothing
      T* const out = (T*)a.out + ((int64_t)(w.first + (real ? mine : 0)) * a.heads + w.kv * group + r_tile % group) * a.size;
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&bar_item_empty[i & 1u]));
      if (some) {
        if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&bar_out[t]), outs++ & 1u, abortp))) {
          if (lane == 0) give_up(48);
          break;
        }
        tc_fence_after();
      }
      auto store8 = [&](int d, const float (&v)[8], float inv) {
        if (!real || d >= a.size) return;
        uint32_t x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = limit > 0 ? pack_pair(v[2 * e] * inv, v[2 * e + 1] * inv, (T*)nullptr) : 0u;
        *(uint4*)(out + d) = make_uint4(x[0], x[1], x[2], x[3]);
      };
      auto inverse = [](float s) { return s > 0.f ? 1.f / s : s == 0.f ? 0.f : s; };  // NaN where a key was
      if (c0 == c1) {
        if (some || j0 == 0) {  // rows that see nothing get their zeros
          const float inv = inverse(sum);
#pragma unroll
          for (int c = 0; c < KD / 32; ++c) {
            uint32_t o[32];
            if (some) {
              tmem_ld32_nowait(o_col + 32 * c, o);
              tmem_ld_wait_for(o);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              float v[8];
#pragma unroll
              for (int x = 0; x < 8; ++x) v[x] = some ? __uint_as_float(o[e * 8 + x]) : 0.f;
              store8(c * 32 + e * 8, v, inv);
            }
          }
          tc_fence_before();
        }
      } else if (some) {
        float* const slot = p.parts + ((size_t)blockIdx.x * 2 + (j0 == 0 ? 1 : 0)) * kPromptPart<KD>;
#pragma unroll
        for (int c = 0; c < KD / 32; ++c) {
          uint32_t o[32];
          tmem_ld32_nowait(o_col + 32 * c, o);
          tmem_ld_wait_for(o);
#pragma unroll
          for (int e = 0; e < 8; ++e) ((uint4*)slot)[(size_t)(c * 8 + e) * 2 * PR_ROWS + r_part] = make_uint4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
        }
        tc_fence_before();
        slot[(size_t)2 * PR_ROWS * KD + r_part] = top;
        slot[(size_t)2 * PR_ROWS * (KD + 1) + r_part] = sum;
        __threadfence();
        asm volatile("bar.sync %0, 128;" ::"r"(1 + t) : "memory");
        if (r_tile == 0) {
          int* const counter = p.counters + c0 * 2 + t;
          last_part[t] = atomicAdd(counter, 1) == c1 - c0;
          if (last_part[t]) *counter = 0;  // nobody else comes: ready for the next launch
        }
        asm volatile("bar.sync %0, 128;" ::"r"(1 + t) : "memory");
        if (last_part[t]) {
          __threadfence();
          auto part_of = [&](int c) { return p.parts + ((size_t)c * 2 + (c == c0 ? 1 : 0)) * kPromptPart<KD>; };
          float all = -INFINITY, total_sum = 0.f;
          for (int c = c0; c <= c1; ++c) all = fmaxf(all, __ldcg(part_of(c) + (size_t)2 * PR_ROWS * KD + r_part));
          for (int c = c0; c <= c1; ++c) {
            const float m = __ldcg(part_of(c) + (size_t)2 * PR_ROWS * KD + r_part);
            if (m != -INFINITY) total_sum += __ldcg(part_of(c) + (size_t)2 * PR_ROWS * (KD + 1) + r_part) * ex2((m - all) * p.slope);
          }
          const float inv = inverse(total_sum);
#pragma unroll 1
          for (int d = 0; d < KD; d += 16) {
            float v[2][8] = {};
#pragma unroll 1
            for (int c = c0; c <= c1; ++c) {
              const float* src = part_of(c);
              const float m = __ldcg(src + (size_t)2 * PR_ROWS * KD + r_part);
              if (m == -INFINITY) continue;
              const float keep = ex2((m - all) * p.slope);
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float4 x = __ldcg((const float4*)src + (size_t)(d / 4 + e) * 2 * PR_ROWS + r_part);
                float* const to = &v[e / 2][e % 2 * 4];
                to[0] += x.x * keep, to[1] += x.y * keep, to[2] += x.z * keep, to[3] += x.w * keep;
              }
            }
            store8(d, v[0], inv);
            store8(d + 8, v[1], inv);
          }
        }
        asm volatile("bar.sync %0, 128;" ::"r"(1 + t) : "memory");  // the word is free again
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

void encode(CUtensorMap* map, const PagedAttention& a, const void* base, int rank, const cuuint64_t* dims, const cuuint64_t* strides, const cuuint32_t* box) {
  const cuuint32_t steps[4] = {1, 1, 1, 1};
  EncodeTiledFn encode = tiled_encoder();
  if (!encode || encode(map, a.dt == DT::F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, rank, const_cast<void*>(base), dims, strides, box, steps,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
    OXB_FAIL("OxiPagedAttention: the driver refused a tensor map");
}
// Boxes of 64 lanes by `box` rows of one head of one page; lanes behind the head and pages behind the cache read as zeros.
void encode_cache(CUtensorMap* map, const PagedAttention& a, const void* cache, int box) {
  const cuuint64_t row = (cuuint64_t)a.kv_heads * a.size * 2;
  const cuuint64_t dims[4] = {(cuuint64_t)a.size, (cuuint64_t)a.kv_heads, (cuuint64_t)a.t.page, (cuuint64_t)a.t.pages}, strides[3] = {(cuuint64_t)a.size * 2, row, row * a.t.page};
  const cuuint32_t boxes[4] = {64, 1, (cuuint32_t)box, 1};
  encode(map, a, cache, 4, dims, strides, boxes);
}
// Boxes of 64 lanes by the query heads of a key head by `span` tokens: the packed rows of a tile, one behind the other.
void encode_queries(CUtensorMap* map, const PagedAttention& a, int span) {
  const cuuint64_t dims[3] = {(cuuint64_t)a.size, (cuuint64_t)a.heads, (cuuint64_t)a.t.tokens}, strides[2] = {(cuuint64_t)a.size * 2, (cuuint64_t)a.heads * a.size * 2};
  const cuuint32_t box[3] = {64, (cuuint32_t)(a.heads / a.kv_heads), (cuuint32_t)span};
  encode(map, a, a.q, 3, dims, strides, box);
}

template <typename T, int KD>
void launch_prompt(const PagedAttention& a, int least_rows, void* workspace, cudaStream_t s) {
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
  const int group = a.heads / a.kv_heads;
  PromptParams p{};
  p.a = a;
  p.parts = (float*)workspace;
  p.counters = (int*)((float*)workspace + (size_t)device_sms() * 2 * kPromptPart<KD>);
  p.box = std::min(a.t.page & -a.t.page, PR_KEYS);  // the largest power of two that divides a page
  p.least_rows = least_rows;
  p.span = PR_ROWS / group;
  encode_queries(&p.queries, a, p.span);
  encode_cache(&p.keys, a, a.key_cache, p.box);
  encode_cache(&p.values, a, a.value_cache, p.box);
  // kind::f16: f32 accumulator, A and B in the cache's type; scores: both K-major, 128 x 128; output: B MN-major, 128 x KD
  const uint32_t type = a.dt == DT::F16 ? 0u : 1u, common = (1u << 4) | (type << 7) | (type << 10) | ((128u >> 4) << 24);
  p.idesc_s = common | ((128u >> 3) << 17);
  p.idesc_o = common | (1u << 16) | (((uint32_t)KD >> 3) << 17);
  p.slope = (a.scale == 0.f ? 1.f : std::fabs(a.scale)) * 1.4426950408889634f;
  p.flip = a.scale < 0.f;
  p.mute = a.scale == 0.f;
  launch(umma_prompt_kernel<T, KD>, dim3(device_sms()), dim3(PR_THREADS), S::kSmem, s, p);
}

}  // namespace

bool paged_attention_prompts_fit(const PagedAttention& a) { return a.size <= 128 && a.heads / a.kv_heads <= PR_ROWS; }

size_t paged_attention_prompts_workspace(const PagedAttention& a) {
  return (size_t)device_sms() * 2 * ((a.size <= 64 ? kPromptPart<64> : kPromptPart<128>) * sizeof(float) + sizeof(int));
}

void paged_attention_prompts(const PagedAttention& a, int least_rows, void* workspace, cudaStream_t s) {
  if (a.dt == DT::F16) a.size <= 64 ? launch_prompt<__half, 64>(a, least_rows, workspace, s) : launch_prompt<__half, 128>(a, least_rows, workspace, s);
  else a.size <= 64 ? launch_prompt<__nv_bfloat16, 64>(a, least_rows, workspace, s) : launch_prompt<__nv_bfloat16, 128>(a, least_rows, workspace, s);
}

}  // namespace k
}  // namespace oxb
