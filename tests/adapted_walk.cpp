// Walks the shares of products with adapters: reads a product a line (row tiles, column tiles, tiles taken whole, blocks of k, adapters of a tile) and says what is
// multiplied more or less than once. Compiled by test_adapted_shares.py.
#include <algorithm>
#include <cstdio>
#include <map>
#include <vector>

using std::max;
using std::min;
#define __host__
#define __device__
#include "shares.cuh"

int main() {
  int row_tiles, column_tiles, shared, k_blocks, adapters, line = 0, bad = 0;
  while (scanf("%d %d %d %d %d", &row_tiles, &column_tiles, &shared, &k_blocks, &adapters) == 5) {
    ++line;
    const int tiles = row_tiles * column_tiles, rest = tiles - shared, extra = row_tiles == 1 ? adapters : 0;
    const int pairs = rest || tiles > PAIRS ? PAIRS : tiles, aligned = rest ? aligned_parts(rest, k_blocks) : 0;
    std::vector<std::vector<int>> k(tiles, std::vector<int>(k_blocks)), a(tiles, std::vector<int>(adapters));
    std::vector<std::map<int, int>> who(tiles);
    for (int pair = 0; pair < pairs; ++pair) {
      Walk walk(pair, pairs, tiles, shared, k_blocks, extra, aligned);
      int t, k0, k1, e0, e1;
      while (walk.next(t, k0, k1, e0, e1)) {
        if (row_tiles > 1) {
          e0 = 0;
          e1 = walk.ends(k0, k1) ? adapters : 0;
        }
        for (int i = k0; i < k1; ++i) ++k[t][i];
        for (int i = e0; i < e1; ++i) ++a[t][i];
        if (t >= shared) {
          ++who[t][pair - walk.first_pair(t)];
          if (walk.count(t) > shares_of_a_tile(rest)) ++bad, printf("line %d: tile %d has %d shares and room for %d\n", line, t, walk.count(t), shares_of_a_tile(rest));
        }
      }
    }
    for (int t = 0; t < tiles; ++t) {
      for (int i = 0; i < k_blocks; ++i)
        if (k[t][i] != 1) ++bad, printf("line %d: tile %d takes block %d of k %d times\n", line, t, i, k[t][i]);
      for (int i = 0; i < adapters; ++i)
        if (a[t][i] != 1) ++bad, printf("line %d: tile %d takes adapter %d %d times\n", line, t, i, a[t][i]);
      if (t < shared) continue;
      const int count = Walk(0, pairs, tiles, shared, k_blocks, extra, aligned).count(t);
      for (int i = 0; i < count; ++i)
        if (who[t][i] != 1) ++bad, printf("line %d: tile %d has share %d %d times\n", line, t, i, who[t][i]);
      if ((int)who[t].size() != count) ++bad, printf("line %d: tile %d counts %d shares and has %zu\n", line, t, count, who[t].size());
    }
  }
  printf("%d products, %d faults\n", line, bad);
  return bad != 0;
}
