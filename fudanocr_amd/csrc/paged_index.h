// Index arithmetic of the paged key / value cache, for the kernels of paged_attention.hip and beam.hip.  Plain C++ with no
// device intrinsics, so that a host program can check every function over whole ranges.
//
// Layout: pages [num_pages][heads][page][dim]; row s of `table` names the pages of sequence s in order; kv_lens[s] tokens are
// in the cache, the new ones included.  All three, and the rows' offsets, come from device memory and are not trusted: a sequence
// whose length does not fit is `bad`, one whose rows do not all lie in the tensors `torn` (its results are NaN in the rows that
// there are, nothing of it is written to the cache) and no address is formed from them.
#pragma once
#ifdef __HIPCC__
#define PG_FN __host__ __device__ __forceinline__
#else
#define PG_FN static inline
#endif

struct PagedShape {
  const int* table;    // [seqs][table_ld]
  const int* kv_lens;  // [seqs]
  const int* q_start;  // [seqs + 1] first row of each sequence's new tokens, or null: `per` rows each
  long tokens, num_pages;
  int seqs, table_ld, page_shift, max_kv;
  int per;             // tokens / seqs where there is no q_start (a 64-bit division is not for every block to do)
};

struct PagedSeq {
  long t0;   // first row of the new tokens
  int n;     // how many
  int len;   // tokens in the cache
  bool bad;  // kv_lens[s] out of range
  bool torn; // its offsets run over the first or the last row
};

// an offset as far as it lies in the tensors (which have less than 2^31 rows)
PG_FN int paged_row(const PagedShape& c, int at) { return at < 0 ? 0 : at > (int)c.tokens ? (int)c.tokens : at; }

// rows of sequence s, as far as they lie in [0, tokens); none where its offsets fall
PG_FN PagedSeq paged_seq(const PagedShape& c, int s) {
  PagedSeq r;
  if (c.q_start) {
    const int a = c.q_start[s], b = c.q_start[s + 1], first = paged_row(c, a), rows = paged_row(c, b) - first;
    r.t0 = first;
    r.n = rows > 0 ? rows : 0;
    r.torn = b > a && (unsigned)rows != (unsigned)b - (unsigned)a;
  } else {
    r.n = c.per;
    r.t0 = (long)s * r.n;
    r.torn = false;
  }
  const int len = c.kv_lens[s];
  r.bad = len < 0 || len > c.max_kv || len > ((long)c.table_ld << c.page_shift);
  r.len = r.bad ? 0 : len;
  return r;
}

// a sequence that gets NaN for its results and writes nothing
PG_FN bool paged_lost(const PagedSeq& q) { return q.bad || q.torn; }

// page that holds position pos of sequence s, or -1 when the table names none
PG_FN int paged_page(const PagedShape& c, int s, int pos) {
  const int p = c.table[(long)s * c.table_ld + (pos >> c.page_shift)];
  return p >= 0 && p < c.num_pages ? p : -1;
}

// keys that new token i of n sees: a prefix of the cache
PG_FN int paged_visible(int len, int n, int i, int causal) {
  const int v = causal ? len - n + 1 + i : len;
  return v < 0 ? 0 : v;
}

// A flat list of row tiles over sequences of unknown lengths: `rows` rows per new token (the heads that share a key), `tile`
// rows per tile.  Sequence s owns the tiles from first(s) on; first(s + 1) - first(s) >= ceil(n * rows / tile) for every
// length, so first(seqs) tiles are enough, and first() is monotone: a tile finds its sequence by search.
PG_FN long paged_first_tile(long t0, int s, int rows, int tile) { return t0 * rows / tile + s; }
PG_FN long paged_tiles(long tokens, int seqs, int rows, int tile) { return tokens * rows / tile + seqs; }
