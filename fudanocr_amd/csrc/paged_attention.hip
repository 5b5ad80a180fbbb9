// Attention of a chunk of new tokens over a paged key / value cache (serving side of the transformer decoders; the cache
// layout and the meaning of its numbers: paged_index.h).  With c = scale, G = heads / kv_heads and the keys j < visible(i):
//   o[i, h] = sum_j p_j v_j / sum_j p_j,   p_j = exp(c q[i, h] . k_j - m),   m = max_j c q[i, h] . k_j
// in one pass over the keys with a running maximum and sum in fp32.
#include "focr_common.h"
#include "paged_index.h"
#include <math.h>

typedef _Float16 f16_t;
typedef __bf16 bf16_t;

__device__ __forceinline__ float pg_to_f(float x) { return x; }
__device__ __forceinline__ float pg_to_f(bf16_t x) { return (float)x; }
__device__ __forceinline__ float pg_to_f(f16_t x) { return (float)x; }

// the last i in [0, n) with f(i) <= key, for a non-decreasing f with f(0) <= key (64 probes a round; all lanes take part)
template <typename F>
__device__ __forceinline__ int pg_find(F f, int n, long key, int lane) {
  int lo = 0;
  while (n > 1) {
    const int step = (n + 63) >> 6, at = lane * step;
    const bool le = at < n && (long)f(lo + at) <= key;
    int k = __popcll(__ballot(le));
    k = k > 0 ? k - 1 : 0;
    lo += k * step;
    n = step < n - k * step ? step : n - k * step;
  }
  return lo;
}

__device__ __forceinline__ int pg_seq_of_row(const PagedShape& c, long t, int lane) {
  if (!c.q_start) return (int)(t / (c.tokens / c.seqs));
  const int* q = c.q_start;
  return pg_find([q](int i) { return q[i]; }, c.seqs, t, lane);
}

// ---- new keys and values into their pages: one wave per token --------------------------------------------------------
template <int UNIT>
__global__ __launch_bounds__(256) void paged_append_kernel(const char* __restrict__ kn, const char* __restrict__ vn, long ldtk,
                                                           long ldhk, long ldtv, long ldhv, char* __restrict__ kp,
                                                           char* __restrict__ vp, PagedShape c, int heads, int row_bytes) {
  const int lane = threadIdx.x & 63;
  const long t = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (t >= c.tokens) return;
  const int s = pg_seq_of_row(c, t, lane);
  const PagedSeq q = paged_seq(c, s);
  const long i = t - q.t0;
  if (q.bad || i < 0 || i >= q.n) return;
  const int pos = q.len - q.n + (int)i;
  if (pos < 0) return;
  const int pg = paged_page(c, s, pos);
  if (pg < 0) return;
  const int slot = pos & ((1 << c.page_shift) - 1), units = row_bytes / UNIT;
  for (int u = lane; u < heads * units; u += 64) {
    const int h = u / units, b = (u - h * units) * UNIT;
    const long dst = ((((long)pg * heads + h) << c.page_shift) + slot) * row_bytes + b;
    const char *ks = kn + t * ldtk + h * ldhk + b, *vs = vn + t * ldtv + h * ldhv + b;
    if (UNIT == 16) {
      const uint4 a = *(const uint4*)ks, w = *(const uint4*)vs;
      *(uint4*)(kp + dst) = a;
      *(uint4*)(vp + dst) = w;
    } else if (UNIT == 4) {
      *(uint32_t*)(kp + dst) = *(const uint32_t*)ks;
      *(uint32_t*)(vp + dst) = *(const uint32_t*)vs;
    } else {
      *(uint16_t*)(kp + dst) = *(const uint16_t*)ks;
      *(uint16_t*)(vp + dst) = *(const uint16_t*)vs;
    }
  }
}

// ---- attention, the plainest form: one wave per (token, head), the head's dimensions across the lanes -----------------
template <typename T, int D>
__global__ __launch_bounds__(256) void paged_attention_row_kernel(const T* __restrict__ q, long ldt, long ldh,
                                                                  const T* __restrict__ kp, const T* __restrict__ vp,
                                                                  PagedShape c, T* __restrict__ o, long ldto, long ldho,
                                                                  int max_q, int heads, int kv_heads, float scale, int causal) {
  constexpr int E = D / 64;
  const int lane = threadIdx.x & 63;
  const long row = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= c.tokens * heads) return;
  const long t = row / heads;
  const int h = (int)(row - t * heads), kh = h / (heads / kv_heads);
  const int s = pg_seq_of_row(c, t, lane);
  const PagedSeq sq = paged_seq(c, s);
  const long i = t - sq.t0;
  if (i < 0 || i >= sq.n) return;
  bool bad = sq.bad || sq.n > max_q;
  float qv[E], acc[E];
  for (int e = 0; e < E; ++e) {
    qv[e] = pg_to_f(q[t * ldt + h * ldh + e * 64 + lane]) * scale;
    acc[e] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  const int vis = bad ? 0 : paged_visible(sq.len, sq.n, (int)i, causal);
  for (int j = 0; j < vis; ++j) {
    const int pg = paged_page(c, s, j);
    if (pg < 0) {
      bad = true;
      break;
    }
    const long at = ((((long)pg * kv_heads + kh) << c.page_shift) + (j & ((1 << c.page_shift) - 1))) * D + lane;
    float d = 0.f;
    for (int e = 0; e < E; ++e) d = fmaf(qv[e], pg_to_f(kp[at + e * 64]), d);
    d = wave_sum(d);
    const float mn = fmaxf(m, d);
    const float base = mn == -INFINITY ? 0.f : mn;
    const float a = expf(m - base), p = expf(d - base);
    m = mn;
    l = l * a + p;
    for (int e = 0; e < E; ++e) acc[e] = acc[e] * a + p * pg_to_f(vp[at + e * 64]);
  }
  for (int e = 0; e < E; ++e)
    o[t * ldto + h * ldho + e * 64 + lane] = (T)(bad ? NAN : l == 0.f ? 0.f : acc[e] / l);
}

// ---- C entries ---------------------------------------------------------------------------------------------------------
static bool pg_shape(PagedShape& c, const int* table, const int* kv_lens, const int* q_start, long tokens, int seqs, int page,
                     int table_ld, long num_pages, int max_kv) {
  if (page < 8 || page > 1024 || (page & (page - 1))) return false;
  c = {table, kv_lens, q_start, tokens, num_pages, seqs, table_ld, __builtin_ctz(page), max_kv};
  return true;
}
static bool pg_aligned(const void* p) { return ((uintptr_t)p & 15) == 0; }
static inline int pg_esize(int dtype) { return dtype == FOCR_DT_F32 ? 4 : 2; }

#define PG_CHECK_COMMON()                                                                                             \
  FOCR_CHECK_ARG(dtype == FOCR_DT_F32 || dtype == FOCR_DT_BF16 || dtype == FOCR_DT_F16, "dtype must be fp32, bf16 or fp16"); \
  FOCR_CHECK_ARG(dim == 64 || dim == 128 || dim == 256, "head dim must be 64, 128 or 256");                           \
  FOCR_CHECK_ARG(tokens >= 0 && tokens <= INT32_MAX && seqs >= 0, "tokens / seqs out of range");                      \
  if (tokens == 0 || seqs == 0) return FOCR_OK;                                                                       \
  FOCR_CHECK_ARG(k_pages && v_pages && table && kv_lens, "null pointer");                                             \
  FOCR_CHECK_ARG(pg_aligned(k_pages) && pg_aligned(v_pages), "pages must be 16-byte aligned");                        \
  FOCR_CHECK_ARG(num_pages > 0 && num_pages <= INT32_MAX && table_ld > 0, "empty cache");                             \
  FOCR_CHECK_ARG(q_start || tokens % seqs == 0, "without q_start every sequence has tokens / seqs rows")

extern "C" int focr_paged_append(const void* k_new, const void* v_new, long ldtk, long ldhk, long ldtv, long ldhv, void* k_pages,
                                 void* v_pages, const int* table, const int* kv_lens, const int* q_start, long tokens, int seqs,
                                 int heads, int dim, int page, int table_ld, long num_pages, int dtype, void* stream) {
  PG_CHECK_COMMON();
  FOCR_CHECK_ARG(k_new && v_new && heads > 0, "null pointer or no heads");
  PagedShape c;
  FOCR_CHECK_ARG(pg_shape(c, table, kv_lens, q_start, tokens, seqs, page, table_ld, num_pages, INT32_MAX),
                 "page must be a power of two from 8 to 1024");
  const long es = pg_esize(dtype);
  const long strides = ldtk | ldhk | ldtv | ldhv;
  const bool wide = pg_aligned(k_new) && pg_aligned(v_new) && ((strides * es) & 15) == 0;
  auto kern = wide ? paged_append_kernel<16> : es == 4 ? paged_append_kernel<4> : paged_append_kernel<2>;
  hipLaunchKernelGGL(kern, dim3(cdiv(tokens, 4)), dim3(256), 0, (hipStream_t)stream, (const char*)k_new, (const char*)v_new,
                     ldtk * es, ldhk * es, ldtv * es, ldhv * es, (char*)k_pages, (char*)v_pages, c, heads, (int)(dim * es));
  FOCR_LAUNCH_CHECK();
  return FOCR_OK;
}

extern "C" long focr_paged_attention_ws_bytes(long tokens, int seqs, int heads, int kv_heads, int dim, int max_q, int max_kv,
                                              int dtype) {
  return 0;
}

extern "C" int focr_paged_attention_fwd(const void* q, long ldt, long ldh, const void* k_pages, const void* v_pages,
                                        const int* table, const int* kv_lens, const int* q_start, void* o, long ldto, long ldho,
                                        void* ws, long ws_bytes, long tokens, int seqs, int heads, int kv_heads, int dim,
                                        int page, int table_ld, long num_pages, int max_q, int max_kv, float scale, int causal,
                                        int dtype, void* stream) {
  PG_CHECK_COMMON();
  FOCR_CHECK_ARG(q && o, "null pointer");
  FOCR_CHECK_ARG(kv_heads > 0 && heads > 0 && heads % kv_heads == 0, "heads must be a multiple of kv_heads");
  FOCR_CHECK_ARG(max_q >= 0 && max_kv >= 0, "max_q / max_kv out of range");
  FOCR_CHECK_ARG(scale > 0.f && scale < INFINITY, "scale must be positive and finite");
  FOCR_CHECK_ARG(q_start || tokens / seqs <= max_q, "max_q is below tokens / seqs");
  PagedShape c;
  FOCR_CHECK_ARG(pg_shape(c, table, kv_lens, q_start, tokens, seqs, page, table_ld, num_pages, max_kv),
                 "page must be a power of two from 8 to 1024");
  const dim3 grid((unsigned)((tokens * heads + 3) / 4));
#define PG_ROW(T, DD)                                                                                                     \
  hipLaunchKernelGGL((paged_attention_row_kernel<T, DD>), grid, dim3(256), 0, (hipStream_t)stream, (const T*)q, ldt, ldh,  \
                     (const T*)k_pages, (const T*)v_pages, c, (T*)o, ldto, ldho, max_q, heads, kv_heads, scale, causal)
#define PG_ROW_D(T)               \
  if (dim == 64) PG_ROW(T, 64);   \
  else if (dim == 128) PG_ROW(T, 128); \
  else PG_ROW(T, 256)
  if (dtype == FOCR_DT_F32) { PG_ROW_D(float); }
  else if (dtype == FOCR_DT_BF16) { PG_ROW_D(bf16_t); }
  else { PG_ROW_D(f16_t); }
  FOCR_LAUNCH_CHECK();
  return FOCR_OK;
}
