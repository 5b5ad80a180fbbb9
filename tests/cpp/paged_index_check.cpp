// CPU check of fudanocr_amd/csrc/paged_index.h (built by tests/test_decode.py with -fsanitize=address,undefined): sequences'
// rows and lengths, page lookups and the flat list of row tiles, for valid numbers and for every kind of bad ones.  The arrays
// are exactly as long as documented, so that the sanitizer sees any read past them.
#include "paged_index.h"
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>

#define REQUIRE(c) do { if (!(c)) { std::printf("FAILED %s:%d %s\n", __FILE__, __LINE__, #c); return 1; } } while (0)

int main() {
  std::mt19937 rng(7);
  auto pick = [&](long lo, long hi) { return std::uniform_int_distribution<long>(lo, hi)(rng); };
  const int junk[] = {-1, INT32_MIN, INT32_MAX, -1000, 1 << 30};
  long checked = 0;
  for (int round = 0; round < 4000; ++round) {
    PagedShape c;
    c.seqs = (int)pick(1, 9);
    c.table_ld = (int)pick(1, 6);
    c.page_shift = (int)pick(3, 10);
    c.num_pages = pick(1, 50);
    c.max_kv = (int)pick(0, ((long)c.table_ld << c.page_shift) + 5);
    std::vector<int> table((size_t)c.seqs * c.table_ld), lens(c.seqs), qs(c.seqs + 1);
    for (int& t : table) t = pick(0, 9) ? (int)pick(0, c.num_pages - 1) : junk[pick(0, 4)];
    for (int& l : lens) l = pick(0, 5) ? (int)pick(0, (long)c.table_ld << c.page_shift) : junk[pick(0, 4)];
    long at = pick(0, 3);
    for (int& q : qs) { q = (int)at; at += pick(0, 3) ? pick(0, 200) : 0; }
    c.tokens = at + pick(0, 4);
    const bool spoilt = pick(0, 4) == 0;
    if (spoilt) qs[pick(0, c.seqs)] = junk[pick(0, 4)];
    c.table = table.data(); c.kv_lens = lens.data(); c.q_start = qs.data();
    if (pick(0, 3) == 0) { c.q_start = nullptr; c.tokens = c.seqs * pick(0, 70); }
    c.per = c.q_start ? 0 : (int)(c.tokens / c.seqs);
    for (int s = 0; s < c.seqs; ++s) {
      const PagedSeq q = paged_seq(c, s);
      REQUIRE(q.n >= 0 && q.t0 >= 0 && q.t0 + q.n <= c.tokens);
      REQUIRE(q.len >= 0 && q.len <= c.max_kv && q.len <= (c.table_ld << c.page_shift));
      REQUIRE(q.bad == (lens[s] < 0 || lens[s] > c.max_kv || lens[s] > (c.table_ld << c.page_shift)));
      for (int pos = 0; pos < q.len; pos += 1 + q.len / 13) {           // every position of a length that passed has a table entry
        const int p = paged_page(c, s, pos);
        const int e = table[(size_t)s * c.table_ld + pos / (1 << c.page_shift)];
        REQUIRE(p == (e >= 0 && e < c.num_pages ? e : -1));
      }
      for (int i = 0; i < q.n; i += 1 + q.n / 7) {
        const int v = paged_visible(q.len, q.n, i, 1);
        REQUIRE(v >= 0 && v <= q.len && (i + 1 < q.n || v == q.len));
        REQUIRE(paged_visible(q.len, q.n, i, 0) == q.len);
      }
    }
    // the flat tile list: every tile of every sequence has a place of its own, in order
    const int rows = (int)pick(1, 9), tile = 16 << pick(0, 4);
    if (!spoilt) {
      long next = 0;
      for (int s = 0; s < c.seqs; ++s) {
        const PagedSeq q = paged_seq(c, s);
        const long f = paged_first_tile(q.t0, s, rows, tile);
        REQUIRE(f >= next);
        next = f + ((long)q.n * rows + tile - 1) / tile;
      }
      REQUIRE(next <= paged_tiles(c.tokens, c.seqs, rows, tile));
      ++checked;
    }
  }
  std::printf("ok %ld\n", checked);
  return 0;
}
