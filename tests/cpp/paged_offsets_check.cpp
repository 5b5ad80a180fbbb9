// CPU check of how fudanocr_amd/csrc/paged_index.h takes offsets that do not fit (built by tests/test_decode.py with
// -fsanitize=address,undefined): ascending ones may begin in front of the first row or end behind the last.  Every row that a
// sequence claims belongs to it alone, the sequence is `torn` exactly if it claims rows that are not there, and the list of row
// tiles holds a place for every tile of the rows that are.
#include "paged_index.h"
#include <cstdint>
#include <cstdio>
#include <random>
#include <vector>

#define REQUIRE(c) do { if (!(c)) { std::printf("FAILED %s:%d %s\n", __FILE__, __LINE__, #c); return 1; } } while (0)

int main() {
  std::mt19937 rng(3);
  auto pick = [&](long lo, long hi) { return std::uniform_int_distribution<long>(lo, hi)(rng); };
  long torn = 0;
  for (int round = 0; round < 20000; ++round) {
    PagedShape c = {};
    c.seqs = (int)pick(1, 9);
    c.table_ld = 1;
    c.page_shift = 3;
    c.num_pages = 1;
    c.max_kv = 8;
    c.tokens = pick(1, 300);
    std::vector<int> table(c.seqs, 0), lens(c.seqs, 8), qs(c.seqs + 1);
    long at = pick(0, 2) ? pick(0, 5) : pick(0, 9) ? -pick(0, 400) : INT32_MIN;
    for (int& q : qs) { q = (int)at; at += pick(0, 3) ? pick(0, 90) : 0; if (!pick(0, 40)) at = INT32_MAX; if (at > INT32_MAX) at = INT32_MAX; }
    c.table = table.data(); c.kv_lens = lens.data(); c.q_start = qs.data();
    std::vector<int> owner(c.tokens, -1);
    const int rows = (int)pick(1, 9), tile = 16 << pick(0, 4);
    long next = 0;
    for (int s = 0; s < c.seqs; ++s) {
      const PagedSeq q = paged_seq(c, s);
      const long claimed = (long)qs[s + 1] - qs[s];
      REQUIRE(!q.bad && q.t0 >= 0 && q.n >= 0 && q.t0 + q.n <= c.tokens && q.n <= claimed);
      REQUIRE(paged_lost(q) == (q.n < claimed));
      torn += q.torn;
      for (long t = 0; t < c.tokens; ++t) {
        const bool mine = t >= qs[s] && t < qs[s + 1];
        REQUIRE(mine == (t >= q.t0 && t < q.t0 + q.n));
        if (mine) { REQUIRE(owner[t] < 0); owner[t] = s; }
      }
      const long first = paged_first_tile(paged_row(c, qs[s]), s, rows, tile);
      REQUIRE(first >= next);
      next = first + ((long)q.n * rows + tile - 1) / tile;
    }
    REQUIRE(next <= paged_tiles(c.tokens, c.seqs, rows, tile));
  }
  REQUIRE(torn > 1000);
  std::printf("ok %ld\n", torn);
  return 0;
}
