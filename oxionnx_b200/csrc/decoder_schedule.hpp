// How the prompt kernel of the paged attention shares its work: plain integer arithmetic, the same on host and device.
//
// A work item is a block of 2 * `span` new tokens of one sequence for one key head (the two tiles of the kernel, `span` tokens
// times the query heads of a key head each), over all its 128-key tiles.  All items' tiles are laid end to end, a sequence's
// blocks in order and the key heads of a block side by side, every item with kBegin steps more for what it costs to begin
// and to end one; a thread block takes an equal run of steps, wherever that cuts an item.
#pragma once

#ifndef OXB_HD
#ifdef __CUDACC__
#define OXB_HD __host__ __device__ __forceinline__
#else
#define OXB_HD inline
#endif
#endif

namespace oxb {
namespace k {

struct PromptWork {
  static constexpr int kKeys = 128;  // of a tile
  // Steps that an item costs beside its tiles.  With 1 / 2 / 3 / 4 of them a prompt of 8192 tokens took 622 / 521 / 489 / 493 us
  // from cold clocks, and warm 556 / 554 with 2 / 3; seven packed ones (209 to 1746 tokens) 183 / 148 / 150 / 164, one of 256
  // tokens 27 / 35 with 2 / 3: blocks with the short items of a prompt's beginning finish late, or early.
  static constexpr int kBegin = 2;

  int rows, base, span, kv_heads;  // new tokens; tokens before them (length - rows, below 0 where rows see nothing); tokens of a tile

  OXB_HD int blocks() const { return (rows + 2 * span - 1) / (2 * span); }
  // key tiles that tile t (0, 1) of block i reads
  OXB_HD int tiles_of(int i, int t) const {
    const long long first = ((long long)i * 2 + t) * span;
    if (first >= rows) return 0;
    const long long seen = (long long)base + (first + span < rows ? first + span : rows);
    return seen <= 0 ? 0 : (int)((seen + kKeys - 1) / kKeys);
  }
  OXB_HD int tiles(int i) const {  // of the item: at least one, in which rows that see nothing get their zeros
    const int a = tiles_of(i, 0), b = tiles_of(i, 1), most = a > b ? a : b;
    return most > 0 ? most : 1;
  }
  OXB_HD int steps(int i) const { return tiles(i) + kBegin; }  // of an item of block i
  // sum of floor((a i + b) / m) over i = 0 .. n - 1, by Euclid's steps on (a, m); a, m up to 2^9, b below 2^32, n below 2^23
  static OXB_HD long long floor_sum(unsigned n, unsigned m, unsigned a, unsigned b) {
    long long sum = 0;
    while (n > 0) {
      sum += (long long)n * (n - 1) / 2 * (a / m) + (long long)n * (b / m);
      a %= m, b %= m;
      const unsigned top = a * n + b;
      if (top < m) break;
      n = top / m, b = top % m;
      const unsigned swap = m;
      m = a, a = swap;
    }
    return sum;
  }
  // steps of the first i blocks of the sequence, all key heads
  OXB_HD long long before(int i) const {
    const int all = blocks(), inner = i < all ? i : all - 1;  // the last block may be short
    long long n = 0;
    if (base >= 0) {
      n = floor_sum((unsigned)inner, kKeys, 2u * span, (unsigned)base + 2u * span + kKeys - 1);
    } else {
      for (int j = 0; j < inner; ++j) n += tiles(j);
    }
    if (i >= all) n += tiles(all - 1);
    return (n + (long long)kBegin * (i < all ? i : all)) * kv_heads;
  }
  OXB_HD long long total() const { return rows > 0 ? before(blocks()) : 0; }
  // The block that step `inside` of the sequence lies in, 32 blocks at a time; what is left of `inside` is the step within it, all
  // key heads.  lanes(steps, inside): of 32 lanes with steps(lane) steps each, the first whose end lies behind `inside`, and the
  // steps of those in front of it; without one, lane 32 and the steps of all.
  struct Found {
    int lane;
    long long before;
  };
  template <typename Lanes>
  OXB_HD int block_of(long long* inside, Lanes&& lanes) const {
    for (int block = 0;; block += 32) {
      const Found f = lanes([&](int lane) { return block + lane < blocks() ? (long long)steps(block + lane) * kv_heads : 0LL; }, *inside);
      *inside -= f.before;
      if (f.lane < 32) return block + f.lane;
      if (block + 32 >= blocks()) return blocks() - 1;  // `inside` is no step of the sequence
    }
  }
  // the same on the host, lane by lane
  OXB_HD int block_at(long long at) const {
    return block_of(&at, [](auto steps, long long inside) {
      Found f{0, 0};
      for (; f.lane < 32 && f.before + steps(f.lane) <= inside; ++f.lane) f.before += steps(f.lane);
      return f;
    });
  }
};

}  // namespace k
}  // namespace oxb
