/* The work list of the prompt kernel (csrc/decoder_schedule.hpp) against a list made item by item: every block of tokens, key
 * head and key tile belongs to exactly one run, the runs' cuts name the same first and last holder of an item as the kernel's
 * arithmetic, and the closed form of the steps before a block is their sum.  Prints "<items> items <bad> bad". */
#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include <vector>

#include "../../oxionnx_b200/csrc/decoder_schedule.hpp"

using oxb::k::PromptWork;

int main(int argc, char** argv) {
  const int rounds = argc > 1 ? atoi(argv[1]) : 200;
  srand(7);
  long items = 0, bad = 0;
  for (int it = 0; it < rounds; ++it) {
    const int group = 1 + rand() % 20, kv_heads = 1 + rand() % 9, runs = 1 + rand() % 200;
    std::vector<PromptWork> sequences(1 + rand() % 6);
    long long total = 0;
    for (PromptWork& w : sequences) {
      w.span = 128 / group, w.kv_heads = kv_heads;
      w.rows = rand() % 5 == 0 ? 0 : 1 + rand() % (it % 3 ? 600 : 5000);
      w.base = rand() % 3 == 0 ? -(rand() % (w.rows + 5)) : rand() % 7000;
      total += w.total();
    }
    if (total == 0) continue;
    const long long per = std::max(6LL, (total + runs - 1) / runs);
    long long at = 0;  // step of the list
    for (const PromptWork& w : sequences) {
      long long inside = 0;
      for (int block = 0; w.rows > 0 && block < w.blocks(); ++block) {
        if (w.before(block) != inside) ++bad;
        for (int kv = 0; kv < kv_heads; ++kv, ++items) {
          const int tiles = w.tiles(block);
          const long long first = at + PromptWork::kBegin;
          const long long c0 = first / per;
          std::vector<int> held(tiles, 0);
          for (long long c = at / per; c <= (first + tiles - 1) / per; ++c) {  // what run c takes of the item
            const long long from = std::max(at, c * per), to = std::min(first + tiles, (c + 1) * per);
            const long long j0 = std::max(0LL, from - first), j1 = to - first;
            if (j1 <= j0) continue;
            for (long long j = j0; j < j1; ++j) ++held[j];
            if ((j0 == 0) != (c == c0)) ++bad;
            for (int t = 0; t < 2; ++t) {  // a tile's parts are those of the runs c0 .. c1, no others
              const int mine = w.tiles_of(block, t);
              const long long c1 = (first + std::max(mine, 1) - 1) / per;
              if (mine > 0 && (j0 < mine) != (c >= c0 && c <= c1)) ++bad;
            }
          }
          for (int h : held) bad += h != 1;
          if (w.block_at(inside) != block || w.block_at(inside + tiles + PromptWork::kBegin - 1) != block) ++bad;
          at += tiles + PromptWork::kBegin, inside += tiles + PromptWork::kBegin;
        }
      }
      if (w.total() != inside) ++bad;
    }
    if (at != total) ++bad;
  }
  printf("%ld items %ld bad\n", items, bad);
  return bad != 0;
}
