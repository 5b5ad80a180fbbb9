// Beam search on the device: the choice of the best continuations over beams and vocabulary, and the reordering of the
// paged caches of the beams that survive.
#include "focr_common.h"
#include "paged_index.h"
#include <math.h>

// ======================================================================================================================
// Selection.  A beam k of a batch entry with running score s_k and logits x_k[0 .. V):
//   candidate (k, v):  c = s_k + x_k[v] - log sum_u exp x_k[u];   a finished beam has one candidate, (k, eos) with c = s_k.
// The n largest in descending order, equal ones in the order of k V + v.  A NaN, and every candidate of a beam whose score or
// normaliser is not finite, ranks as -inf.  Continuations of different beams may differ by less than fp32 resolves, so the
// normaliser and the comparison are held in 64 bits; the scores that go out are rounded once.
// ======================================================================================================================
__device__ __forceinline__ float bs_load(const void* p, long i, int dtype) {
  if (dtype == FOCR_DT_F32) return ((const float*)p)[i];
  if (dtype == FOCR_DT_BF16) return (float)((const __bf16*)p)[i];
  return (float)((const _Float16*)p)[i];
}
struct BsBest {
  double c;
  long i;
};
__device__ __forceinline__ bool bs_before(double ca, long ia, double cb, long ib) { return ca > cb || (ca == cb && ia < ib); }

__global__ __launch_bounds__(256) void beam_select_kernel(const void* __restrict__ logits, long ldb, long ldk,
                                                          const float* __restrict__ scores, const uint8_t* __restrict__ fin,
                                                          float* __restrict__ out_scores, int* __restrict__ out_parents,
                                                          long long* __restrict__ out_tokens, uint8_t* __restrict__ out_fin,
                                                          int beams, int vocab, int n, int eos, int dtype) {
  __shared__ double add[64];          // s_k - normaliser; NaN: the beam is dead
  __shared__ BsBest best[4];
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  for (int k = wave; k < beams; k += 4) {
    const long row = b * ldb + k * ldk;
    float m = -INFINITY;
    bool nan = false;
    for (int v = lane; v < vocab; v += 64) {
      const float x = bs_load(logits, row + v, dtype);
      nan |= x != x;
      m = fmaxf(m, x);
    }
    m = wave_max(m);
    nan = __ballot(nan) != 0;
    double sum = 0.0;
    for (int v = lane; v < vocab; v += 64) sum += exp((double)bs_load(logits, row + v, dtype) - (double)m);
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
    const float s = scores[b * beams + k];
    double a = (double)s - ((double)m + log(sum));
    if (fin && fin[b * beams + k]) a = (double)s;
    else if (nan || !isfinite(m)) a = NAN;
    if (!isfinite(s)) a = NAN;
    if (lane == 0) add[k] = a;
  }
  __syncthreads();
  double pc = INFINITY;
  long pi = -1;
  const long total = (long)beams * vocab;
  for (int r = 0; r < n; ++r) {
    double bc = -INFINITY;
    long bi = INT64_MAX;
    for (long i = tid; i < total; i += 256) {
      const int k = (int)(i / vocab), v = (int)(i - (long)k * vocab);
      double c;
      if (fin && fin[b * beams + k]) c = v == eos ? add[k] : (double)-INFINITY;
      else c = add[k] + (double)bs_load(logits, b * ldb + k * ldk + v, dtype);
      if (!(c == c)) c = -INFINITY;
      if (bs_before(pc, pi, c, i) && bs_before(c, i, bc, bi)) bc = c, bi = i;
    }
    for (int o = 32; o > 0; o >>= 1) {
      const double c = __shfl_xor(bc, o, 64);
      const long i = __shfl_xor(bi, o, 64);
      if (bs_before(c, i, bc, bi)) bc = c, bi = i;
    }
    if (lane == 0) best[wave] = {bc, bi};
    __syncthreads();
    pc = best[0].c, pi = best[0].i;
    for (int w = 1; w < 4; ++w)
      if (bs_before(best[w].c, best[w].i, pc, pi)) pc = best[w].c, pi = best[w].i;
    __syncthreads();
    if (tid == 0) {
      const int k = (int)(pi / vocab), v = (int)(pi - (long)k * vocab);
      out_scores[b * n + r] = (float)pc;
      out_parents[b * n + r] = k;
      out_tokens[b * n + r] = v;
      out_fin[b * n + r] = (fin && fin[b * beams + k]) || v == eos;
    }
  }
}

extern "C" long focr_beam_select_ws_bytes(int batch, int beams, int vocab, int n, int dtype) { return 0; }

extern "C" int focr_beam_select(const void* logits, long ldb, long ldk, const float* scores, const uint8_t* finished,
                                float* out_scores, int* out_parents, long long* out_tokens, uint8_t* out_finished, void* ws,
                                long ws_bytes, int batch, int beams, int vocab, int n, int eos, int dtype, void* stream) {
  FOCR_CHECK_ARG(dtype == FOCR_DT_F32 || dtype == FOCR_DT_BF16 || dtype == FOCR_DT_F16, "dtype must be fp32, bf16 or fp16");
  FOCR_CHECK_ARG(batch >= 0 && beams > 0 && beams <= 64 && vocab > 0, "beams must be 1 to 64, vocab positive");
  FOCR_CHECK_ARG(n > 0 && n <= 64 && n <= (long)beams * vocab, "n must be 1 to 64 and at most beams * vocab");
  FOCR_CHECK_ARG(!finished || (eos >= 0 && eos < vocab), "finished beams need an eos inside the vocabulary");
  if (batch == 0) return FOCR_OK;
  FOCR_CHECK_ARG(logits && scores && out_scores && out_parents && out_tokens && out_finished, "null pointer");
  hipLaunchKernelGGL(beam_select_kernel, dim3(batch), dim3(256), 0, (hipStream_t)stream, logits, ldb, ldk, scores, finished,
                     out_scores, out_parents, out_tokens, out_finished, beams, vocab, n, eos, dtype);
  FOCR_LAUNCH_CHECK();
  return FOCR_OK;
}

// ======================================================================================================================
// Reordering.  The beams of a group have the same length L; beam j goes on from beam p = parents[j].  Full pages are never
// written again, so j takes p's table entries for them.  The last, partial page (L % page tokens) will be written by every
// beam: a j != p gets its own copy, in its spare page, and the page it held before becomes its spare.  So a beam moves at most
// page - 1 tokens however long the sequence, and no page is allocated or freed.
// ======================================================================================================================
#define BR_MAX_TENSORS 64
struct BrPages {
  char* p[BR_MAX_TENSORS];
};

__device__ __forceinline__ int br_parent(const int* parents, int slot, int beams) {
  const int p = parents[slot];
  return p >= 0 && p < beams ? slot / beams * beams + p : slot;          // no such beam: the slot goes on from itself
}

// grid (16 KB pieces of a page, slot, tensor)
__global__ __launch_bounds__(256) void beam_copy_pages_kernel(BrPages pages, const int* __restrict__ parents,
                                                              const int* __restrict__ table, const int* __restrict__ lens,
                                                              const int* __restrict__ spare, int beams, int heads,
                                                              int row_units, int page_shift, int table_ld, long num_pages) {
  const int slot = blockIdx.y, src_slot = br_parent(parents, slot, beams);
  if (src_slot == slot) return;
  const int len = lens[slot / beams * beams], full = len >> page_shift, rest = len & ((1 << page_shift) - 1);
  if (len < 0 || full >= table_ld || rest == 0) return;
  const int from = table[(long)src_slot * table_ld + full], to = spare[slot];
  if (from < 0 || from >= num_pages || to < 0 || to >= num_pages) return;
  const int run = rest * row_units, total = heads * run;                 // 16-byte units
  const long head_units = (long)row_units << page_shift;
  uint4* base = (uint4*)pages.p[blockIdx.z];
  const uint4* s = base + (long)from * heads * head_units;
  uint4* d = base + (long)to * heads * head_units;
  const int x0 = blockIdx.x * 1024 + threadIdx.x;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int x = x0 + i * 256;
    if (x < total) {
      const int h = x / run;
      const long at = h * head_units + (x - h * run);
      d[at] = s[at];
    }
  }
}

// one thread per table column of a group: it reads the column of every beam before it writes one, so the outputs may be the
// inputs
__global__ __launch_bounds__(256) void beam_tables_kernel(const int* __restrict__ parents, const int* table,
                                                          const int* __restrict__ lens, const int* spare, int* table_out,
                                                          int* spare_out, int beams, int page_shift, int table_ld) {
  extern __shared__ int br_col[];                                        // [beams][256]
  const int g = blockIdx.y, col = blockIdx.x * 256 + threadIdx.x, first = g * beams;
  if (col >= table_ld) return;
  const int len = lens[first], full = len >> page_shift, rest = len & ((1 << page_shift) - 1);
  const bool ok = len >= 0 && (full < table_ld || (full == table_ld && rest == 0));
  for (int k = 0; k < beams; ++k) br_col[k * 256 + threadIdx.x] = table[(long)(first + k) * table_ld + col];
  for (int k = 0; k < beams; ++k) {
    const int slot = first + k, p = ok ? br_parent(parents, slot, beams) : slot, own = br_col[k * 256 + threadIdx.x];
    const bool partial = ok && rest && col == full;
    int e = own;
    if (ok && col < full) e = br_col[(p - first) * 256 + threadIdx.x];
    else if (partial && p != slot) e = spare[slot];
    table_out[(long)slot * table_ld + col] = e;
    if (partial) spare_out[slot] = p != slot ? own : spare[slot];
    else if (col == 0 && !(ok && rest)) spare_out[slot] = spare[slot];   // nothing partial in this group
  }
}

extern "C" int focr_beam_reorder(const int* parents, const int* table, const int* kv_lens, const int* spare, int* table_out,
                                 int* spare_out, void* const* pages, int tensors, int groups, int beams, int heads, int dim,
                                 int page, int table_ld, long num_pages, int dtype, void* stream) {
  FOCR_CHECK_ARG(dtype == FOCR_DT_F32 || dtype == FOCR_DT_BF16 || dtype == FOCR_DT_F16, "dtype must be fp32, bf16 or fp16");
  FOCR_CHECK_ARG(groups >= 0 && beams > 0 && beams <= 64 && (long)groups * beams <= 65535, "beams must be 1 to 64, slots at most 65535");
  FOCR_CHECK_ARG(page >= 8 && page <= 1024 && !(page & (page - 1)), "page must be a power of two from 8 to 1024");
  FOCR_CHECK_ARG(heads > 0 && dim > 0 && tensors >= 0 && table_ld > 0 && num_pages > 0, "empty cache");
  const long row_bytes = (long)dim * (dtype == FOCR_DT_F32 ? 4 : 2), page_bytes = heads * (row_bytes * page);
  FOCR_CHECK_ARG(row_bytes % 16 == 0 && page_bytes <= (1l << 30), "rows must be whole 16-byte units, a page at most 1 GB");
  if (groups == 0) return FOCR_OK;
  FOCR_CHECK_ARG(parents && table && kv_lens && spare && table_out && spare_out && (pages || !tensors), "null pointer");
  for (int i = 0; i < tensors; ++i) FOCR_CHECK_ARG(pages[i] && ((uintptr_t)pages[i] & 15) == 0, "pages must be 16-byte aligned");
  const int shift = __builtin_ctz(page);
  for (int i = 0; i < tensors; i += BR_MAX_TENSORS) {
    BrPages b = {};
    const int m = tensors - i < BR_MAX_TENSORS ? tensors - i : BR_MAX_TENSORS;
    for (int j = 0; j < m; ++j) b.p[j] = (char*)pages[i + j];
    hipLaunchKernelGGL(beam_copy_pages_kernel, dim3(cdiv(page_bytes, 16384), groups * beams, m), dim3(256), 0,
                       (hipStream_t)stream, b, parents, table, kv_lens, spare, beams, heads, (int)(row_bytes / 16), shift,
                       table_ld, num_pages);
    FOCR_LAUNCH_CHECK();
  }
  hipLaunchKernelGGL(beam_tables_kernel, dim3(cdiv(table_ld, 256), groups), dim3(256), beams * 1024, (hipStream_t)stream,
                     parents, table, kv_lens, spare, table_out, spare_out, beams, shift, table_ld);
  FOCR_LAUNCH_CHECK();
  return FOCR_OK;
}
