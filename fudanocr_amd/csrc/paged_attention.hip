// Attention of a chunk of new tokens over a paged key / value cache (serving side of the transformer decoders; the cache
// layout and the meaning of its numbers: paged_index.h).  With c = scale, G = heads / kv_heads and the keys j < visible(i):
//   o[i, h] = sum_j p_j v_j / sum_j p_j,   p_j = exp(c q[i, h] . k_j - m),   m = max_j c q[i, h] . k_j
// in one pass over the keys with a running maximum and sum in fp32.
#include "focr_common.h"
#include "paged_index.h"
#include <math.h>

typedef _Float16 f16_t;
typedef __bf16 bf16_t;

typedef unsigned long long u64_mask;

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
  if (!c.q_start) return (int)t / c.per;
  const int* q = c.q_start;
  return pg_find([q](int i) { return q[i]; }, c.seqs, t, lane);
}

// ---- new keys and values into their pages: one wave per token, 16 bytes a lane where the rows allow it.  A launch's latency (4 us
// for 64 tokens) up to some thousand tokens ----------------------------------------------------------------------------
template <int UNIT>
__global__ __launch_bounds__(256) void paged_append_kernel(const char* __restrict__ kn, const char* __restrict__ vn, long ldtk,
                                                           long ldhk, long ldtv, long ldhv, char* __restrict__ kp,
                                                           char* __restrict__ vp, PagedShape c, int heads, int row_bytes) {
  const int lane = threadIdx.x & 63;
  const long t = (long)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (t >= c.tokens) return;
  const int s = pg_seq_of_row(c, t, lane);
  const PagedSeq q = paged_seq(c, s);
  const long i = t - q.t0;
  if (paged_lost(q) || i < 0 || i >= q.n) return;
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

// ---- matrix instructions -----------------------------------------------------------------------------------------------
// Operands are 16-byte chunks of a row: 8 16-bit or 4 fp32 values of the contraction axis.  Lane l of a 16 x 16 tile holds row
// l % 16 of A (column l % 16 of B) at chunk l / 16, lane l of the 32 x 32 tile row l % 32 at chunk l / 32; any order of the
// contraction axis will do as long as A and B share it.  Results: column l % 16, rows 4 (l / 16) + i, or column l % 32, rows
// 8 (i / 4) + 4 (l / 32) + i % 4.  fp32 runs on the exact fp32 instructions, one value of the chunk at a time.
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(4))) uint32_t u32x4;
template <typename T> struct PgMma;
template <> struct PgMma<bf16_t> {
  static __device__ __forceinline__ f32x4 mma16(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(focr_bf16x8, a), __builtin_bit_cast(focr_bf16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x16 mma32(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(focr_bf16x8, a), __builtin_bit_cast(focr_bf16x8, b), c, 0, 0, 0);
  }
  static constexpr uint32_t EXP = 0x7f80u, ONE = 0x3f80u;
};
template <> struct PgMma<f16_t> {
  static __device__ __forceinline__ f32x4 mma16(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x16 mma32(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
  static constexpr uint32_t EXP = 0x7c00u, ONE = 0x3c00u;
};
template <> struct PgMma<float> {
  static __device__ __forceinline__ f32x4 mma16(u32x4 a, u32x4 b, f32x4 c) {
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[i]), __uint_as_float(b[i]), c, 0, 0, 0);
    return c;
  }
  static __device__ __forceinline__ f32x16 mma32(u32x4 a, u32x4 b, f32x16 c) {
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a[i]), __uint_as_float(b[i]), c, 0, 0, 0);
    return c;
  }
  static constexpr uint32_t EXP = 0x7f800000u, ONE = 0x3f800000u;
};

// two fp32 values as a 16-bit pair, rounded to nearest: the weights p lie in [0, 1] relative to the running maximum, so a
// weight loses at most half a step of the output's own type and the errors of a row's keys average out
template <typename T> __device__ __forceinline__ uint32_t pg_pack(float a, float b);
template <> __device__ __forceinline__ uint32_t pg_pack<bf16_t>(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, focr_bf16x2));
}
template <> __device__ __forceinline__ uint32_t pg_pack<f16_t>(float a, float b) {
  typedef __attribute__((ext_vector_type(2))) _Float16 f16x2;
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, f16x2));
}

// a word of values with its infinities and NaN replaced by zero
template <typename T> __device__ __forceinline__ uint32_t pg_finite(uint32_t w) {
  if constexpr (sizeof(T) == 4) return (w & 0x7f800000u) == 0x7f800000u ? 0u : w;
  const uint32_t e = PgMma<T>::EXP;
  if ((w & e) == e) w &= 0xffff0000u;
  if ((w >> 16 & e) == e) w &= 0xffffu;
  return w;
}
// one where a chunk holds +inf (CLS 1), -inf (2) or NaN (3), zero elsewhere
template <typename T, int CLS> __device__ __forceinline__ u32x4 pg_class(u32x4 a) {
  u32x4 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 4) {
      const uint32_t w = a[i];
      r[i] = (CLS == 1 ? w == 0x7f800000u : CLS == 2 ? w == 0xff800000u : (w & 0x7fffffffu) > 0x7f800000u) ? 0x3f800000u : 0u;
    } else {
      uint32_t out = 0;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t w = a[i] >> (16 * h) & 0xffffu, e = PgMma<T>::EXP;
        const bool hit = CLS == 1 ? w == e : CLS == 2 ? w == (e | 0x8000u) : (w & 0x7fffu) > e;
        out |= (hit ? PgMma<T>::ONE : 0u) << (16 * h);
      }
      r[i] = out;
    }
  }
  return r;
}
// what a sum of p v becomes when it also holds `pos` values +inf, `neg` values -inf and `nan` NaN
__device__ __forceinline__ float pg_with_nonfinite(float x, float pos, float neg, float nan) {
  if (pos > 0.f) x += INFINITY;
  if (neg > 0.f) x -= INFINITY;
  return nan > 0.f ? NAN : x;
}

// exp2(c2 (s - mx)), ref = c2 mx (0 when there is no maximum yet).  One multiply-add; in fp32, where the matrix instructions
// leave time, from the difference, which loses nothing near the maximum.  fp16 weights are taken 2^14 times as large, sums and all:
// a long tail of weights below fp16's 6e-8 would count in the sum (fp32) and not in the product
template <typename T> __device__ __forceinline__ float pg_weight(float s, float c2, float mx, float ref) {
  if constexpr (sizeof(T) == 4) return __builtin_amdgcn_exp2f((s - (mx == -INFINITY ? 0.f : mx)) * c2);
  else return __builtin_amdgcn_exp2f(fmaf(s, c2, (PgMma<T>::EXP == 0x7c00u ? 14.f : 0.f) - ref));
}

// What the weights of a row are relative to, as its sums are kept and joined: the maximum itself in fp32, `ref` (the rounded
// product, which every weight was taken against) in the 16-bit types.  Two of them are compared by their difference, so that sums
// whose maximum stands are multiplied by 1 exactly: c2 m - ref in one multiply-add is the rounding error of c2 m there, once for
// every other row of the wave that finds a new maximum, always with the same sign
template <typename T> __device__ __forceinline__ float pg_top(float mx, float c2) { return sizeof(T) == 4 ? mx : mx * c2; }
template <typename T> __device__ __forceinline__ float pg_ratio(float top, float to, float c2) {       // `to` above -inf
  return __builtin_amdgcn_exp2f(sizeof(T) == 4 ? (top - to) * c2 : top - to);
}
// a running sum's factor when its maximum goes from m to mx; ref = c2 mx rounded, either 0 while there is no maximum
template <typename T> __device__ __forceinline__ float pg_rescale(float m, float mx, float c2, float ref) {
#pragma clang fp contract(off)
  if constexpr (sizeof(T) == 4) return __builtin_amdgcn_exp2f((m - (mx == -INFINITY ? 0.f : mx)) * c2);
  else return __builtin_amdgcn_exp2f(m * c2 - ref);
}

// a part's sum of weights at maximum `top` relative to the common one; a part without keys has sum 0 at maximum -inf, one whose
// scores are all NaN has a NaN sum there, which must not get lost
template <typename T> __device__ __forceinline__ float pg_share(float sum, float top, float to, float c2) {
  return sum == 0.f ? 0.f : sum != sum ? sum : sum * pg_ratio<T>(top, to, c2);
}

template <typename T>
struct PgArgs {
  const T* q;
  long ldt, ldh;
  const T *kp, *vp;
  PagedShape c;
  T* o;
  long ldto, ldho;
  float* part;   // [split][token][head][D], weights relative to the split's own maximum
  float2* ml;    // [split][token][head]: that maximum (pg_top) and the sum of the weights
  int max_q, heads, kv_heads, group, nsplit, chunk, tile_chunk, tiles, causal, thin_rows, wide_q, wide_o;
  float c2;      // scale * log2(e)
};

template <typename T, int N> __device__ __forceinline__ void pg_store_row(T* p, const float (&v)[N], bool wide) {
  if (wide) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < N; i += 4) *(f32x4*)(p + i) = f32x4{v[i], v[i + 1], v[i + 2], v[i + 3]};
    } else {
      uint32_t w[N / 2];
#pragma unroll
      for (int i = 0; i < N / 2; ++i) w[i] = pg_pack<T>(v[2 * i], v[2 * i + 1]);
      if constexpr (N == 8) *(u32x4*)p = u32x4{w[0], w[1], w[2], w[3]};
      else *(uint2*)p = uint2{w[0], w[1]};
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) p[i] = (T)v[i];
  }
}

// 16-byte chunk of a query row
template <typename T> __device__ __forceinline__ u32x4 pg_load_chunk(const T* p, bool wide) {
  if (wide) return *(const u32x4*)p;
  if constexpr (sizeof(T) == 4) {
    return u32x4{__float_as_uint(p[0]), __float_as_uint(p[1]), __float_as_uint(p[2]), __float_as_uint(p[3])};
  } else {
    const uint16_t* w = (const uint16_t*)p;
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = w[2 * i] | (uint32_t)w[2 * i + 1] << 16;
    return r;
  }
}

// rows of a sequence whose numbers do not fit: NaN
template <typename T, int D>
__device__ __forceinline__ void pg_fill_nan(const PgArgs<T>& a, const PagedSeq& sq, int kh, int threads) {
  const long total = (long)sq.n * a.group * D;
  for (long i = threadIdx.x; i < total; i += threads) {
    const long r = i / D;
    a.o[(sq.t0 + r / a.group) * a.ldto + (kh * a.group + r % a.group) * a.ldho + i % D] = (T)NAN;
  }
}

// ======================================================================================================================
// Few rows (one token, or a few tokens and the heads that share a key head: up to 16 NT rows), a long axis of keys: bound by
// the bytes of the keys and values, which are read once, straight into registers in the matrix instructions' own layout -- no
// LDS, no barrier in the loop, 4 waves a block that take every fourth tile of KT keys and are joined at the end.
//   S^T = K Q^T   A = 16 keys x chunk (lane: key l % 16, chunk l / 16 + 4 u), B = queries from registers;
//   O^T = V^T P^T  the lane that holds column q of S^T holds the weights of keys 4 (l / 16) + i: already B's layout when the
//                 contraction index means those keys.  A = V^T needs, per lane, these keys' values at ONE d: the lane loads the
//                 NK keys' rows at d = CH (l % 16) .. + CH (16 lanes = whole row, coalesced) and transposes its NK x CH square in
//                 registers (v_perm, 16-bit types; a choice of registers in fp32); tile (u, c) of O^T then has row e <-> d =
//                 16 CH u + CH e + c.
// The next tile's loads go out between the two products.  MFMA time is a tenth of the bytes' (16-bit) to a third (fp32).
// Measured: 64 sequences of 100 .. 8190 tokens, 8 key heads x 128 bf16: 173 us = 5.7 TB/s; two of 131 000: 177 us = 6.1 TB/s; 128
// images x 256 positions, 16 heads x 64 fp32: 43 us = 6.4 TB/s (a large copy on this card: 4.9 TB/s read and written).  32 rows a key
// head (32 sequences x 4 tokens over 4000, 4 key heads x 128), per call: bf16 61 us = 4.3 TB/s, fp32 131 us = 4.0.
// ======================================================================================================================
#define PG_MAX_CHUNK 8192
// Queries that take 32 registers or more go through LDS.  At most 256 registers keep two waves on a SIMD; 16-bit rows of 256
// (106 us, spilling at two waves 132: 32 sequences of 4000 tokens, 4 key heads) and 32 rows x 256 take one
template <typename T, int D, int NT> constexpr bool pg_thin_q_lds() { return NT * D * sizeof(T) >= 512; }
template <typename T, int D, int NT> constexpr int pg_thin_waves() {
  return NT * D <= 64 ? 4 : D == 256 && (NT == 2 || sizeof(T) == 2) ? 1 : 2;
}
template <typename T, int D, int NT>
__global__ __launch_bounds__(256, (pg_thin_waves<T, D, NT>())) void paged_thin_kernel(PgArgs<T> a) {
  constexpr int ES = sizeof(T), EC = 16 / ES;          // elements of a chunk
  constexpr int NU = D * ES / 64;                      // chunk quads of a row (S^T contraction steps)
  constexpr int NK = ES == 4 ? 4 : 8, KT = 4 * NK;     // keys of a lane, keys of a tile
  constexpr int CH = (D / 16 < EC) ? D / 16 : EC, VU = D / (16 * CH);  // values of one V load, loads per row
  constexpr int PITCH = D + 4;
  __shared__ int pages[PG_MAX_CHUNK / 8 + 2];
  __shared__ float red[16 * NT * PITCH];
  __shared__ float2 wml[4][16 * NT];
  constexpr bool QLDS = pg_thin_q_lds<T, D, NT>();
  __shared__ u32x4 qs[QLDS ? NT * NU * 64 : 1];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l16 = lane & 15, g = lane >> 4;
  const PagedShape& c = a.c;
  // splits in the slowest place: blocks go round the 8 XCDs by number, and the last splits of most sequences are empty
  const int kh = blockIdx.x % a.kv_heads, s = blockIdx.x / a.kv_heads % c.seqs, split = blockIdx.x / a.kv_heads / c.seqs;
  const PagedSeq sq = paged_seq(c, s);
  if (sq.n * a.group > a.thin_rows && sq.n <= a.max_q) return;           // the other kernel's
  if (sq.n == 0) return;
  if (paged_lost(sq) || sq.n > a.max_q) {
    if (split == 0 && (sq.n <= a.max_q || a.thin_rows >= a.max_q * a.group)) pg_fill_nan<T, D>(a, sq, kh, 256);
    return;
  }
  const int R = sq.n * a.group;
  const int vmin = paged_visible(sq.len, sq.n, 0, a.causal), kend = paged_visible(sq.len, sq.n, sq.n - 1, a.causal);
  const int k0 = split * a.chunk;
  const bool direct = sq.len <= a.chunk;
  if (split && k0 >= kend) return;
  const int k1 = kend < k0 + a.chunk ? kend : k0 + a.chunk;

  // page numbers of this block's keys; one that names no page makes every row NaN
  int any_bad = 0;
  const int p0 = k0 >> c.page_shift, np = k1 > k0 ? ((k1 - 1) >> c.page_shift) - p0 + 1 : 0;
  for (int i = tid; i < np; i += 256) {
    const int p = paged_page(c, s, (p0 + i) << c.page_shift);
    any_bad |= p < 0;
    pages[i] = p < 0 ? 0 : p;
  }

  u32x4 qf[QLDS ? 1 : NT][QLDS ? 1 : NU];
  int vis[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int r = t * 16 + l16;
    const bool ok = r < R;
    const int i = ok ? r / a.group : 0, h = kh * a.group + (ok ? r - i * a.group : 0);
    vis[t] = ok ? paged_visible(sq.len, sq.n, i, a.causal) : 0;
    const T* p = a.q + (sq.t0 + i) * a.ldt + h * a.ldh + g * EC;
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      if (QLDS && (u & 3) != wave) continue;
      const u32x4 x = ok ? pg_load_chunk(p + u * 4 * EC, a.wide_q) : u32x4{0, 0, 0, 0};
      if constexpr (QLDS) qs[(t * NU + u) * 64 + lane] = x;
      else qf[t][u] = x;
    }
  }
  any_bad = __syncthreads_or(any_bad);
  auto q_chunk = [&](int t, int u) {
    if constexpr (QLDS) return qs[(t * NU + u) * 64 + lane];
    else return qf[t][u];
  };

  const long head_bytes = ((long)D * ES) << c.page_shift, page_bytes = head_bytes * a.kv_heads;
  const char *kbase = (const char*)a.kp + kh * head_bytes, *vbase = (const char*)a.vp + kh * head_bytes;
  const int slot_mask = (1 << c.page_shift) - 1;
  u32x4 kr[KT / 16][NU];
  uint32_t vr[NK][VU * CH * ES / 4];
  auto row_at = [&](int key) { return pages[(key >> c.page_shift) - p0] * page_bytes + (long)(key & slot_mask) * (D * ES); };
  auto load_k = [&](int base) {
#pragma unroll
    for (int sub = 0; sub < KT / 16; ++sub) {
      const int key = base + sub * 16 + l16;
      const char* p = kbase + row_at(key < k1 ? key : k1 - 1) + g * 16;
#pragma unroll
      for (int u = 0; u < NU; ++u) kr[sub][u] = *(const u32x4*)(p + u * 64);
    }
  };
  auto load_v = [&](int base) {
#pragma unroll
    for (int qd = 0; qd < NK / 4; ++qd) {
      // four keys that lie in one page; behind the last key: the quad that holds it (its tail may never have been written)
      const int key = base + qd * 16 + 4 * g, last = (k1 - 1) & ~3;
      const char* p = vbase + row_at(key < last ? key : last) + l16 * (CH * ES);
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int u = 0; u < VU; ++u) {
          const char* w = p + j * (D * ES) + u * (16 * CH * ES);
          if constexpr (CH * ES == 16) {
            const u32x4 x = *(const u32x4*)w;
#pragma unroll
            for (int e = 0; e < 4; ++e) vr[qd * 4 + j][u * 4 + e] = x[e];
          } else {
            const uint2 x = *(const uint2*)w;
            vr[qd * 4 + j][u * 2] = x.x;
            vr[qd * 4 + j][u * 2 + 1] = x.y;
          }
        }
    }
  };
  // A operand of O^T's tile (u, cc): this lane's keys at d = 16 CH u + CH (l % 16) + cc
  auto v_frag = [&](int u, int cc) {
    u32x4 r;
    if constexpr (ES == 4) {
#pragma unroll
      for (int j = 0; j < 4; ++j) r[j] = vr[j][u * CH + cc];
    } else {
      const int w = (u * CH + cc) / 2;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        r[j] = __builtin_amdgcn_perm(vr[2 * j + 1][w], vr[2 * j][w], (cc & 1) ? 0x07060302u : 0x05040100u);
    }
    return r;
  };

  f32x4 acc[NT][VU][CH];
  float m[NT], l[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    m[t] = -INFINITY;
    l[t] = 0.f;
#pragma unroll
    for (int u = 0; u < VU; ++u)
#pragma unroll
      for (int e = 0; e < CH; ++e) acc[t][u][e] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  int base = k0 + wave * KT;
  if (base < k1) {
    load_k(base);
    load_v(base);
  }
  for (; base < k1; base += 4 * KT) {
    const int next = base + 4 * KT;
    f32x4 sc[NT][KT / 16];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int sub = 0; sub < KT / 16; ++sub) {
        sc[t][sub] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int u = 0; u < NU; ++u) sc[t][sub] = PgMma<T>::mma16(kr[sub][u], q_chunk(t, u), sc[t][sub]);
      }
    if (next < k1) load_k(next);
    if (base + KT > vmin) {
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int sub = 0; sub < KT / 16; ++sub)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (base + sub * 16 + 4 * g + i >= vis[t]) sc[t][sub][i] = -INFINITY;
    }
    u32x4 pf[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      float mx = m[t];
#pragma unroll
      for (int sub = 0; sub < KT / 16; ++sub)
#pragma unroll
        for (int i = 0; i < 4; ++i) mx = fmaxf(mx, sc[t][sub][i]);
      mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
      mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
      const float ref = mx == -INFINITY ? 0.f : mx * a.c2;
      if (__any(mx > m[t])) {
        const float al = pg_rescale<T>(m[t], mx, a.c2, ref);
        l[t] *= al;
#pragma unroll
        for (int u = 0; u < VU; ++u)
#pragma unroll
          for (int e = 0; e < CH; ++e) acc[t][u][e] *= al;
        m[t] = mx;
      }
      float p[KT / 4];
#pragma unroll
      for (int sub = 0; sub < KT / 16; ++sub)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          p[sub * 4 + i] = pg_weight<T>(sc[t][sub][i], a.c2, mx, ref);
          l[t] += p[sub * 4 + i];
        }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (ES == 4) pf[t][j] = __float_as_uint(p[j]);
        else pf[t][j] = pg_pack<T>(p[2 * j], p[2 * j + 1]);
      }
    }
    if (base + KT > k1) {                              // behind the last key: whatever the page holds must not count
#pragma unroll
      for (int j = 0; j < NK; ++j)
        if (base + (j / 4) * 16 + 4 * g + (j & 3) >= k1) {
#pragma unroll
          for (int w = 0; w < VU * CH * ES / 4; ++w) vr[j][w] = 0;
        }
    }
    bool odd = false;                                  // 0 * inf: values that some of the rows do not see
    if (base + KT > vmin && vmin < kend) {
#pragma unroll
      for (int j = 0; j < NK; ++j)
#pragma unroll
        for (int w = 0; w < VU * CH * ES / 4; ++w) odd |= pg_finite<T>(vr[j][w]) != vr[j][w];
      odd = __any(odd);
    }
    if (odd) {
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        u32x4 see;                                     // one where this lane's key is visible to its row
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if constexpr (ES == 4) see[j] = base + 4 * g + j < vis[t] ? 0x3f800000u : 0u;
          else {
            const int key = base + (j / 2) * 16 + 4 * g + (2 * j & 3);
            see[j] = (key < vis[t] ? PgMma<T>::ONE : 0u) | (key + 1 < vis[t] ? PgMma<T>::ONE << 16 : 0u);
          }
        }
#pragma unroll
        for (int u = 0; u < VU; ++u)
#pragma unroll
          for (int e = 0; e < CH; ++e) {
            const u32x4 vf = v_frag(u, e);
            const f32x4 z = {0.f, 0.f, 0.f, 0.f};
            const f32x4 pos = PgMma<T>::mma16(pg_class<T, 1>(vf), see, z), neg = PgMma<T>::mma16(pg_class<T, 2>(vf), see, z);
            const f32x4 nan = PgMma<T>::mma16(pg_class<T, 3>(vf), see, z);
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[t][u][e][i] = pg_with_nonfinite(acc[t][u][e][i], pos[i], neg[i], nan[i]);
            __builtin_amdgcn_sched_barrier(0);         // one tile at a time: this path must not cost the others registers
          }
      }
#pragma unroll
      for (int j = 0; j < NK; ++j)
#pragma unroll
        for (int w = 0; w < VU * CH * ES / 4; ++w) vr[j][w] = pg_finite<T>(vr[j][w]);
    }
#pragma unroll
    for (int u = 0; u < VU; ++u)
#pragma unroll
      for (int e = 0; e < CH; ++e) {
        const u32x4 vf = v_frag(u, e);
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[t][u][e] = PgMma<T>::mma16(vf, pf[t], acc[t][u][e]);
        if (NT * D >= 256 && (e & 1)) __builtin_amdgcn_sched_barrier(0);       // no more transposed chunks ahead than registers
      }
    if (next < k1) load_v(next);
  }

  // join the waves: one common maximum, then the sums one wave after the other (a fixed order)
  const int nw = k1 - k0 > 3 * KT ? 4 : k1 - k0 > 2 * KT ? 3 : k1 - k0 > KT ? 2 : 1;
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    l[t] += __shfl_xor(l[t], 16, 64);
    l[t] += __shfl_xor(l[t], 32, 64);
    if (g == 0) wml[wave][t * 16 + l16] = float2{pg_top<T>(m[t], a.c2), l[t]};
  }
  __syncthreads();
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    float mx = wml[0][t * 16 + l16].x;
    for (int w = 1; w < nw; ++w) mx = fmaxf(mx, wml[w][t * 16 + l16].x);
    const float al = m[t] == -INFINITY ? 0.f : pg_ratio<T>(pg_top<T>(m[t], a.c2), mx, a.c2);
    for (int w = 0; w < nw; ++w) {
      if (w == wave) {
#pragma unroll
        for (int u = 0; u < VU; ++u)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            f32x4* p = (f32x4*)&red[(t * 16 + l16) * PITCH + u * 16 * CH + (4 * g + i) * CH];
#pragma unroll
            for (int e = 0; e < CH; e += 4) {
              f32x4 v = {acc[t][u][e][i] * al, acc[t][u][e + 1][i] * al, acc[t][u][e + 2][i] * al, acc[t][u][e + 3][i] * al};
              if (w) v += p[e / 4];
              p[e / 4] = v;
            }
          }
      }
      __syncthreads();
    }
  }
  constexpr int N = ES == 4 ? 4 : 8;
  for (int x = tid; x < R * (D / N); x += 256) {
    const int r = x / (D / N), d = (x - r * (D / N)) * N, i = r / a.group, h = kh * a.group + r - i * a.group;
    float mx = wml[0][r].x, ls = 0.f;
    for (int w = 1; w < nw; ++w) mx = fmaxf(mx, wml[w][r].x);
    for (int w = 0; w < nw; ++w) ls += pg_share<T>(wml[w][r].y, wml[w][r].x, mx, a.c2);
    if (any_bad) ls = NAN;
    float v[N];
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = red[r * PITCH + d + e];
    if (direct) {
      const float inv = ls == 0.f ? 0.f : 1.f / ls;
#pragma unroll
      for (int e = 0; e < N; ++e) v[e] = ls == 0.f ? 0.f : v[e] * inv;
      pg_store_row<T, N>(a.o + (sq.t0 + i) * a.ldto + h * a.ldho + d, v, a.wide_o);
    } else {
      const long row = ((long)split * c.tokens + sq.t0 + i) * a.heads + h;
#pragma unroll
      for (int e = 0; e < N; e += 4) *(f32x4*)(a.part + row * D + d + e) = f32x4{v[e], v[e + 1], v[e + 2], v[e + 3]};
      if (d == 0) a.ml[row] = float2{any_bad ? 0.f : mx, ls};
    }
  }
}

// ======================================================================================================================
// Many rows (a chunk's tokens x the heads that share a key head, flattened: a block takes 32 NW neighbouring rows, so one
// staged tile of keys serves every head of the group): bound by the matrix instructions.  32 x 32 tiles in the same
// orientation as above -- S^T = K Q^T leaves a lane one query column, whose weights are B of O^T = V^T P^T as they stand -- with
// KT keys and values at a time in LDS, double-buffered by direct loads, 16-byte chunks XOR-swizzled by row so that both the
// row-wise reads of K and the transposing reads of V (ds_read_b64_tr_b16; plain words in fp32) use every bank.  A wave skips
// the tiles that none of its rows sees and compares positions only where its rows differ.
// Measured: 4096 tokens after 12288, 32 heads over 8, 128 bf16: 0.96 ms = 1000 TFLOP/s (0.97 .. 1.0 ms a call, box to box), where a
// large library product of the same type reaches 1104; the matrix pipe is 0.45 busy and the vector pipe (the exponentials, above all)
// 0.52: two waves a SIMD run as the sum of the two.  fp32 rows of 64 / 128 / 256: 86 / 111 / 82 TFLOP/s on the exact instructions
// (library product: 151); fp16 rows of 64: 592, bf16 rows of 256, which spill: 521.
// ======================================================================================================================
template <int CPR> __device__ __forceinline__ int pg_swz(int row) {
  if constexpr (CPR == 8) return ((row >> 1 & 1) << 2) | ((row >> 2 & 1) << 1) | (row >> 3 & 1);
  else return ((row & 7) << 1) | (row >> 3 & 1);
}
typedef __attribute__((ext_vector_type(4))) short pg_s16x4;
__device__ __forceinline__ uint2 pg_read_tr(const char* p) {
  return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) pg_s16x4*)p));
}

template <typename T, int D, int NW> constexpr int pg_tile_waves() { return NW == 8 || D * sizeof(T) <= 512 ? 2 : 1; }
template <typename T, int D, int NW>
__global__ __launch_bounds__(64 * NW, (pg_tile_waves<T, D, NW>())) void paged_tile_kernel(PgArgs<T> a) {
  constexpr int ES = sizeof(T), EC = 16 / ES, ROWB = D * ES, CPR = ROWB / 16;
  constexpr int KT = ROWB <= 256 ? 64 : 32, NS = KT / 32;
  constexpr int NU = ROWB / 32;                        // contraction steps of S^T (pairs of chunks)
  constexpr int RPI = 64 / CPR;                        // rows one direct load of a wave brings
  constexpr int NL = KT / (RPI * NW);                  // such loads per wave, for K and for V
  constexpr int DT = D / 32, PT = ES == 4 ? 4 : 2;     // O^T tiles; contraction steps of O^T per 32 keys
  constexpr int ROWS = 32 * NW;
  extern __shared__ __attribute__((aligned(128))) char pg_smem[];
  char* const ksm = pg_smem;                           // [2][KT][ROWB]
  char* const vsm = pg_smem + 2 * KT * ROWB;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l32 = lane & 31, hh = lane >> 5;
  const PagedShape& c = a.c;
  const int kh = blockIdx.x % a.kv_heads, split = blockIdx.x / a.kv_heads / a.tiles;
  const int turn = blockIdx.x / a.kv_heads % a.tiles;
  // The tiles with the most keys first, so that the last blocks to finish are short ones.  Up to 64 sequences are put in order of
  // their lengths by the wave itself (24 chunks of 1 .. 764 tokens behind 300 .. 4000: 205 us so, 216 us in the order of the rows;
  // with the priorities below 188); more of them fill the card well enough from the last row to the first.
  int s, tile;
  if (c.seqs <= 64) {
    int len = 0, mine = 0, start = 0;
    if (lane < c.seqs) {
      const PagedSeq sq = paged_seq(c, lane);
      len = sq.len;
      if (sq.n * a.group > a.thin_rows) mine = (sq.n * a.group + ROWS - 1) / ROWS;
    }
    for (int j = 0; j < c.seqs; ++j) {
      const int lj = __builtin_amdgcn_readlane(len, j), tj = __builtin_amdgcn_readlane(mine, j);
      if (lj > len || (lj == len && j < lane)) start += tj;
    }
    const u64_mask hit = __ballot(turn >= start && turn - start < mine);
    if (!hit) return;
    s = __builtin_ctzll(hit);
    tile = __builtin_amdgcn_readlane(mine, s) - 1 - (turn - __builtin_amdgcn_readlane(start, s));
  } else {
    const int* qs = c.q_start;
    const long n = c.per, at = a.tiles - 1 - turn;
    const int grp = a.group;
    auto first = [&](int i) { return paged_first_tile(qs ? (long)paged_row(c, qs[i]) : i * n, i, grp, ROWS); };
    s = pg_find(first, c.seqs, at, lane);
    tile = (int)(at - first(s));
  }
  const PagedSeq sq = paged_seq(c, s);
  const int R = sq.n * a.group, r0 = tile * ROWS;      // (the host has checked that tokens x heads and a tile more fit)
  if (tile < 0 || r0 >= R || R <= a.thin_rows) return;
  if (paged_lost(sq) || sq.n > a.max_q) {
    if (split == 0)
      for (int x = tid; x < ROWS * D; x += 64 * NW) {
        const int r = r0 + x / D;
        if (r < R) a.o[(sq.t0 + r / a.group) * a.ldto + (kh * a.group + r % a.group) * a.ldho + x % D] = (T)NAN;
      }
    return;
  }
  const int tok0 = r0 / a.group, tok1 = (R < r0 + ROWS ? R - 1 : r0 + ROWS - 1) / a.group;
  const int vmin = paged_visible(sq.len, sq.n, tok0, a.causal), kend = paged_visible(sq.len, sq.n, tok1, a.causal);
  const bool direct = sq.len <= a.tile_chunk;
  const int k0 = split * a.tile_chunk;
  if (split && k0 >= kend) return;
  const int k1 = kend < k0 + a.tile_chunk ? kend : k0 + a.tile_chunk;
  const int nt = k1 > k0 ? (k1 - k0 + KT - 1) / KT : 0;

  // this wave's rows: one query column per lane
  u32x4 qf[NU];
  const int row = r0 + wave * 32 + l32;
  const bool ok = row < R;
  const int tok = ok ? row / a.group : 0, head = kh * a.group + (ok ? row - tok * a.group : 0);
  const int vis = ok ? paged_visible(sq.len, sq.n, tok, a.causal) : 0;
  int wvmin = ok ? vis : INT32_MAX, wvmax = vis;
  const T* p = a.q + (sq.t0 + tok) * a.ldt + head * a.ldh + hh * EC;
#pragma unroll
  for (int u = 0; u < NU; ++u) qf[u] = ok ? pg_load_chunk(p + u * 2 * EC, a.wide_q) : u32x4{0, 0, 0, 0};
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const int x = __shfl_xor(wvmin, o, 64), y = __shfl_xor(wvmax, o, 64);
    wvmin = x < wvmin ? x : wvmin;
    wvmax = y > wvmax ? y : wvmax;
  }
  wvmin = __builtin_amdgcn_readfirstlane(wvmin);
  wvmax = __builtin_amdgcn_readfirstlane(wvmax);

  const long head_bytes = (long)ROWB << c.page_shift, page_bytes = head_bytes * a.kv_heads;
  const char *kbase = (const char*)a.kp + kh * head_bytes, *vbase = (const char*)a.vp + kh * head_bytes;
  const int slot_mask = (1 << c.page_shift) - 1;
  const int* trow = c.table + (long)s * c.table_ld;
  int pg[NL];
  bool bad_page = false;
  auto key_of = [&](int base, int i) {                 // key this lane brings in load i; past the end: the last one again
    const int k = base + (i * NW + wave) * RPI + lane / CPR;
    return k < k1 ? k : k1 - 1;
  };
  auto find_pages = [&](int base) {
#pragma unroll
    for (int i = 0; i < NL; ++i) pg[i] = trow[key_of(base, i) >> c.page_shift];
  };
  auto stage = [&](int base, int buf) {
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int row = (i * NW + wave) * RPI + lane / CPR;
      const bool ok = (uint32_t)pg[i] < (uint32_t)c.num_pages;
      bad_page |= !ok;
      const long at = (ok ? pg[i] : 0) * page_bytes + (long)(key_of(base, i) & slot_mask) * ROWB
                      + (((lane % CPR) ^ pg_swz<CPR>(row)) * 16);
      const int dst = buf * KT * ROWB + (i * NW + wave) * 1024;
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(kbase + at),
                                       (__attribute__((address_space(3))) void*)(ksm + dst), 16, 0, 0);
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(vbase + at),
                                       (__attribute__((address_space(3))) void*)(vsm + dst), 16, 0, 0);
    }
  };
  // LDS offsets.  Rows enter the swizzle by their last four bits, of which a lane's row fixes all but constants of the unrolled
  // loops: a few lane offsets, the rest are immediate (left to itself the compiler keeps every address and spills them)
  constexpr bool LEAN = CPR > 16;                      // wide rows: one offset and an xor per read, the registers are short
  constexpr int NKB = LEAN ? 1 : CPR == 8 ? 4 : 8;     // chunk pairs up to the width of the swizzle
  constexpr int NVB = LEAN ? 1 : CPR == 8 ? 2 : 4;     // the same in O^T tiles (16-bit types)
  int koff[NKB], voff[2][NVB];
#pragma unroll
  for (int j = 0; j < NKB; ++j) koff[j] = l32 * ROWB + (((2 * j + hh) ^ pg_swz<CPR>(l32)) << 4);
  const int vrow = hh * 4 + (lane >> 2 & 3), vchunk = (lane >> 4 & 1) * 2 + (lane >> 1 & 1);
#pragma unroll
  for (int e = 0; e < 2; ++e)
#pragma unroll
    for (int j = 0; j < NVB; ++j)
      voff[e][j] = (vrow + e * 8) * ROWB + (((4 * j + vchunk) ^ pg_swz<CPR>(vrow + e * 8)) << 4) + (lane & 1) * 8;
  // A operand of O^T: 32 values d of the keys sub * 32 + step * (32 / PT) ..
  auto v_frag = [&](const char* v, int sub, int step, int dt) {
    u32x4 r;
    if constexpr (ES == 4) {
      const int lane_at = ((l32 >> 2) ^ (hh * 8)) << 4;            // swizzle of row 4 hh; the rest is one xor per word
#pragma unroll
      for (int e = 0; e < 4; ++e)
        r[e] = *(const uint32_t*)(v + (lane_at ^ (((dt & 1) * 8) ^ (e * 2) ^ (step & 1)) << 4) + hh * 4 * ROWB + (l32 & 3) * 4
                                  + (sub * 32 + step * 8 + e) * ROWB + (dt >> 1) * 256);
    } else {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const char* at = LEAN ? v + (voff[e][0] ^ (dt & 3) << 6) + dt / 4 * 256 : v + voff[e][dt % NVB] + dt / NVB * 256;
        const uint2 x = pg_read_tr(at + (sub * 32 + step * 16) * ROWB);
        r[2 * e] = x.x;
        r[2 * e + 1] = x.y;
      }
    }
    return r;
  };

  f32x16 acc[DT];
  float m = -INFINITY, l = 0.f;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) acc[dt] = f32x16{0};
  if (nt) {
    find_pages(k0);
    stage(k0, 0);
    find_pages(k0 + KT < k1 ? k0 + KT : k0);
  }
  for (int it = 0; it < nt; ++it) {
    const int base = k0 + it * KT, buf = it & 1;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();                                   // this tile is there; everyone is done with the other buffer
    if (it + 1 < nt) {
      stage(base + KT, buf ^ 1);
      find_pages(base + 2 * KT < k1 ? base + 2 * KT : k0);
    }
    const char *kt = ksm + buf * KT * ROWB, *vt = vsm + buf * KT * ROWB;
    bool odd = false;
    if (base + KT > vmin) {                            // some row of the block does not see all of this tile: 0 * inf
      char* mine = (char*)vt + tid * 16;
#pragma unroll
      for (int i = 0; i < KT * ROWB / (1024 * NW); ++i) {
        const u32x4 x = *(const u32x4*)(mine + i * 1024 * NW);
#pragma unroll
        for (int w = 0; w < 4; ++w) odd |= pg_finite<T>(x[w]) != x[w];
      }
      odd = __syncthreads_or(odd);
      if (odd) {
        // what the infinities and NaN of the tile add to the rows that see them; then they leave the tile
#pragma unroll 1
        for (int sub = 0; sub < NS; ++sub)
#pragma unroll 1
          for (int step = 0; step < PT; ++step) {
            u32x4 see;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              if constexpr (ES == 4) see[j] = base + sub * 32 + step * 8 + hh * 4 + j < vis ? PgMma<T>::ONE : 0u;
              else {
                const int key = base + sub * 32 + step * 16 + (j >> 1) * 8 + hh * 4 + (2 * j & 3);
                see[j] = (key < vis ? PgMma<T>::ONE : 0u) | (key + 1 < vis ? PgMma<T>::ONE << 16 : 0u);
              }
            }
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
              const u32x4 vf = v_frag(vt, sub, step, dt);
              const f32x16 z = {0};
              const f32x16 pos = PgMma<T>::mma32(pg_class<T, 1>(vf), see, z);
#pragma unroll
              for (int i = 0; i < 16; ++i) acc[dt][i] = pg_with_nonfinite(acc[dt][i], pos[i], 0.f, 0.f);
              const f32x16 neg = PgMma<T>::mma32(pg_class<T, 2>(vf), see, z);
#pragma unroll
              for (int i = 0; i < 16; ++i) acc[dt][i] = pg_with_nonfinite(acc[dt][i], 0.f, neg[i], 0.f);
              const f32x16 nan = PgMma<T>::mma32(pg_class<T, 3>(vf), see, z);
#pragma unroll
              for (int i = 0; i < 16; ++i) acc[dt][i] = pg_with_nonfinite(acc[dt][i], 0.f, 0.f, nan[i]);
              __builtin_amdgcn_sched_barrier(0);
            }
          }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < KT * ROWB / (1024 * NW); ++i) {
          u32x4 x = *(const u32x4*)(mine + i * 1024 * NW);
#pragma unroll
          for (int w = 0; w < 4; ++w) x[w] = pg_finite<T>(x[w]);
          *(u32x4*)(mine + i * 1024 * NW) = x;
        }
        __syncthreads();
      }
    }
    if (base >= wvmax) continue;                       // nothing here for this wave's rows
    f32x16 sc[NS];
#pragma unroll
    for (int sub = 0; sub < NS; ++sub) {
      sc[sub] = f32x16{0};
#pragma unroll
      for (int u = 0; u < NU; ++u) {
        const char* at = LEAN ? kt + (koff[0] ^ (u & 7) << 5) + u / 8 * 256 : kt + koff[u % NKB] + u / NKB * 256;
        const u32x4 kf = *(const u32x4*)(at + sub * 32 * ROWB);
        sc[sub] = PgMma<T>::mma32(kf, qf[u], sc[sub]);
      }
    }
    // The softmax of one wave ahead of the products of its neighbour on the SIMD, while two blocks of 4 waves share a CU (the 24
    // chunks: 204 -> 188 us); in one block of 8 it costs 2 %
    if constexpr (NW == 4) __builtin_amdgcn_s_setprio(1);
    if (base + KT > wvmin) {
#pragma unroll
      for (int sub = 0; sub < NS; ++sub)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (base + sub * 32 + 8 * (i >> 2) + 4 * hh + (i & 3) >= vis) sc[sub][i] = -INFINITY;
    }
    u32x4 pf[NS][PT];
    float mx = m;
#pragma unroll
    for (int sub = 0; sub < NS; ++sub)
#pragma unroll
      for (int i = 0; i < 16; ++i) mx = fmaxf(mx, sc[sub][i]);
    mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
    const float ref = mx == -INFINITY ? 0.f : mx * a.c2;
    if (__any(mx > m)) {
      const float al = pg_rescale<T>(m, mx, a.c2, ref);
      l *= al;
      // what the tile's infinities have added stays also where what came before goes: by the smallest number there is, not by 0
      const float keep = odd && al == 0.f ? 0x1p-149f : al;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) acc[dt] *= keep;
      m = mx;
    }
#pragma unroll
    for (int sub = 0; sub < NS; ++sub) {
      float p[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        p[i] = pg_weight<T>(sc[sub][i], a.c2, mx, ref);
        l += p[i];
      }
#pragma unroll
      for (int step = 0; step < PT; ++step)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if constexpr (ES == 4) pf[sub][step][j] = __float_as_uint(p[step * 4 + j]);
          else pf[sub][step][j] = pg_pack<T>(p[step * 8 + 2 * j], p[step * 8 + 2 * j + 1]);
        }
    }
    if constexpr (NW == 4) __builtin_amdgcn_s_setprio(0);
#pragma unroll
    for (int sub = 0; sub < NS; ++sub)
#pragma unroll
      for (int step = 0; step < PT; ++step)
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          const u32x4 vf = v_frag(vt, sub, step, dt);
          acc[dt] = PgMma<T>::mma32(vf, pf[sub][step], acc[dt]);
        }
  }
  const bool any_bad = __syncthreads_or(bad_page);

  // out: lane = row, four neighbouring values d = 32 dt + 8 q + 4 (l / 32) + ..
  float ls = l + __shfl_xor(l, 32, 64);
  if (any_bad) ls = NAN;
  if (!ok) return;
  const float inv = direct ? (ls == 0.f ? 0.f : 1.f / ls) : 1.f;
  T* o = a.o + (sq.t0 + tok) * a.ldto + head * a.ldho + 4 * hh;
  const long out_row = ((long)split * c.tokens + sq.t0 + tok) * a.heads + head;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      float v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = ls == 0.f ? 0.f : acc[dt][4 * q + e] * inv;
      if (direct) pg_store_row<T, 4>(o + dt * 32 + q * 8, v, a.wide_o);
      else *(f32x4*)(a.part + out_row * D + dt * 32 + q * 8 + 4 * hh) = f32x4{v[0], v[1], v[2], v[3]};
    }
  if (!direct && hh == 0) a.ml[out_row] = float2{any_bad ? 0.f : pg_top<T>(m, a.c2), ls};
}

// ---- joins the splits of a row.  WPR waves of a block of 4 share a (token, head): 1 where rows are many and splits few, 4 where
// a long cache was cut into dozens (69 000 rows, 4 splits: 51 us with a block each, most of it for starting blocks) ----------
template <typename T, int D, int WPR>
__global__ __launch_bounds__(256) void paged_join_kernel(PgArgs<T> a) {
  constexpr int E = D / 64;
  __shared__ float wmax[4], wsum[4], acc[3][D];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), part = wave % WPR;
  const long rows = a.c.tokens * a.heads;
  const int row = blockIdx.x * (4 / WPR) + wave / WPR;
  if (row >= rows) return;                             // (with 4 waves a row there is no such row)
  const int t = row / a.heads, h = row - t * a.heads, s = pg_seq_of_row(a.c, t, lane);
  const PagedSeq sq = paged_seq(a.c, s);
  const long i = t - sq.t0;
  const int chunk = sq.n * a.group <= a.thin_rows ? a.chunk : a.tile_chunk;
  if (i < 0 || i >= sq.n || paged_lost(sq) || sq.n > a.max_q || sq.len <= chunk) return;
  const int n = (paged_visible(sq.len, sq.n, (int)i, a.causal) + chunk - 1) / chunk;
  float mx = -INFINITY;
  for (int k = part * 64 + lane; k < n; k += 64 * WPR) mx = fmaxf(mx, a.ml[row + k * rows].x);
  mx = wave_max(mx);
  if constexpr (WPR == 4) {
    if (lane == 0) wmax[wave] = mx;
    __syncthreads();
    mx = fmaxf(fmaxf(wmax[0], wmax[1]), fmaxf(wmax[2], wmax[3]));
  }
  float ls = 0.f, v[E];
#pragma unroll
  for (int e = 0; e < E; ++e) v[e] = 0.f;
#pragma unroll 4
  for (int k = part; k < n; k += WPR) {
    const float2 ml = a.ml[row + k * rows];
    const float w = ml.x == -INFINITY ? 0.f : pg_ratio<T>(ml.x, mx, a.c2);
    ls += pg_share<T>(ml.y, ml.x, mx, a.c2);
    const float* p = a.part + (row + k * rows) * D + lane * E;
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] += w * p[e];
  }
  if constexpr (WPR == 4) {
    if (lane == 0) wsum[wave] = ls;
    if (wave)
      for (int e = 0; e < E; ++e) acc[wave - 1][lane * E + e] = v[e];
    __syncthreads();
    if (wave) return;
    ls = wsum[0] + wsum[1] + wsum[2] + wsum[3];
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] += acc[0][lane * E + e] + acc[1][lane * E + e] + acc[2][lane * E + e];
  }
  T* o = a.o + t * a.ldto + h * a.ldho + lane * E;
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = (T)(ls == 0.f ? 0.f : v[e] / ls);
}

// ---- C entries ---------------------------------------------------------------------------------------------------------
static bool pg_shape(PagedShape& c, const int* table, const int* kv_lens, const int* q_start, long tokens, int seqs, int page,
                     int table_ld, long num_pages, int max_kv) {
  if (page < 8 || page > 1024 || (page & (page - 1))) return false;
  c = {table, kv_lens, q_start, tokens, num_pages, seqs, table_ld, __builtin_ctz(page), max_kv, q_start ? 0 : (int)(tokens / seqs)};
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
  FOCR_CHECK_ARG(tokens >> 26 == 0, "too many tokens for one launch");
  PagedShape c;
  FOCR_CHECK_ARG(pg_shape(c, table, kv_lens, q_start, tokens, seqs, page, table_ld, num_pages, INT32_MAX),
                 "page must be a power of two from 8 to 1024");
  const long es = pg_esize(dtype), cache = num_pages * heads * page * dim * es;
  const long kb = ((tokens - 1) * ldtk + (heads - 1) * ldhk + dim) * es, vb = ((tokens - 1) * ldtv + (heads - 1) * ldhv + dim) * es;
  FOCR_CHECK_ARG(!focr_overlap(k_pages, cache, v_pages, cache), "k_pages and v_pages share memory");
  FOCR_CHECK_ARG(!focr_overlap(k_new, kb, k_pages, cache) && !focr_overlap(k_new, kb, v_pages, cache) &&
                     !focr_overlap(v_new, vb, k_pages, cache) && !focr_overlap(v_new, vb, v_pages, cache),
                 "the new tokens share memory with the cache");
  const long strides = ldtk | ldhk | ldtv | ldhv;
  const bool wide = pg_aligned(k_new) && pg_aligned(v_new) && ((strides * es) & 15) == 0;
  auto kern = wide ? paged_append_kernel<16> : es == 4 ? paged_append_kernel<4> : paged_append_kernel<2>;
  hipLaunchKernelGGL(kern, dim3(cdiv(tokens, 4)), dim3(256), 0, (hipStream_t)stream, (const char*)k_new, (const char*)v_new,
                     ldtk * es, ldhk * es, ldtv * es, ldhv * es, (char*)k_pages, (char*)v_pages, c, heads, (int)(dim * es));
  FOCR_LAUNCH_CHECK();
  return FOCR_OK;
}

// Splits of the key axis.  The keys of a (sequence, key head) go to blocks of `chunk` keys; a sequence of at most `chunk` keys
// writes its output directly, the parts of a longer one are joined by a second launch.  (Times here compare the forms as they were
// when the rule was made.)  Up to 4096 blocks, so that sequences
// of very different lengths still fill the card evenly (64 sequences of 100 .. 8190 tokens x 8 heads, bf16, 128 wide: 2048
// blocks 198 us, 4096 193 us, 8192 200 us), but no fewer than 1024 keys in a block while there are blocks enough for two on each
// CU: a block's start and end cost as much as some hundred keys (2 sequences of 131k: 1024 keys 205 us, 512 224 us, 256 254 us).
//
// Calls with longer chunks go to the tile kernel, 128 rows a block.
//   * Split over keys only when there are fewer than two such blocks a CU (24 chunks of 1 .. 764 tokens x 32 heads, bf16, 85 tiles x
//     8 key heads: 221 us unsplit, 232 / 240 us cut for 1024 / 2048 blocks: the parts are written and read in fp32), into 1024 keys
//     or more (1024 tokens alone, 32 heads: 37 us, in halves 48), fewer only when that leaves half of the CUs idle (4 chunks of 64
//     behind 1000, fp32: 54 us, in halves 85).
//   * 256 rows a block halve the reads from LDS per product, but make one block a CU: taken when 128-row blocks would fill the
//     card twice over and sequences are long (4096 tokens after 12288: 1058 -> 948 us; the 24 chunks: 221 -> 250 us).
//   * In a ragged call that has mostly short sequences those go to the thin kernel in a launch of their own; with 32 rows a
//     sequence or more on average the tiles take them along (the 24 chunks, 11 of them single tokens: 303 -> 221 us).
struct PgPlan {
  int thin_rows;           // sequences of at most this many rows go to the thin kernel, the rest to the tiles
  int nsplit, chunk;       // of the thin kernel
  int tsplit, tile_chunk;  // of the tiles
  int tile_waves;          // 32 rows each
};
static PgPlan pg_plan(long tokens, int seqs, int kv_heads, int group, int max_q, int max_kv, bool ragged) {
  PgPlan p = {0, 1, 128, 1, INT32_MAX, 4};
  const long rmax = (long)max_q * group;
  if (rmax <= 32) p.thin_rows = rmax <= 16 ? 16 : 32;
  else if (ragged && tokens * group <= 32l * seqs) p.thin_rows = group <= 16 ? 16 : group <= 32 ? 32 : 0;
  if (p.thin_rows) {
    const long groups = (long)seqs * kv_heads, want = (4096 + groups - 1) / groups;
    long chunk = (max_kv + want - 1) / want;
    if (chunk < 1024) chunk = 1024;
    if (groups * ((max_kv + chunk - 1) / chunk) < 512) {
      chunk = max_kv * groups / 512;
      chunk = chunk < 256 ? 256 : chunk > 1024 ? 1024 : chunk;
    }
    chunk = (chunk + 127) / 128 * 128;
    if (chunk > PG_MAX_CHUNK) chunk = PG_MAX_CHUNK;
    const int n = (int)((max_kv + chunk - 1) / chunk);
    p.nsplit = n > 0 ? n : 1;
    p.chunk = (int)chunk;
  }
  if (rmax > 32) {
    const long blocks = (tokens * group + 127) / 128 * kv_heads;
    if (blocks < 512 && max_kv > 512) {
      long chunk = max_kv * blocks / 512;
      if (chunk < 1024) chunk = 1024;
      if (blocks * ((max_kv + chunk - 1) / chunk) < 256) chunk = max_kv * blocks / 256;
      if (chunk < 256) chunk = 256;
      if (chunk < max_kv) {
        p.tsplit = (int)((max_kv + chunk - 1) / chunk);
        p.tile_chunk = (int)(((max_kv + p.tsplit - 1) / p.tsplit + 127) / 128 * 128);
      }
    }
    if (blocks >= 1024 && tokens * group >= 1024l * seqs) p.tile_waves = 8;
  }
  return p;
}
static long pg_ws_bytes(const PgPlan& p, long rows, int dim) {
  const long n = p.nsplit > p.tsplit ? p.nsplit : p.tsplit;
  return n == 1 ? 0 : n * rows * (dim + 2) * 4;
}

// the larger of the two forms (one or several row counts per call) is asked for
extern "C" long focr_paged_attention_ws_bytes(long tokens, int seqs, int heads, int kv_heads, int dim, int max_q, int max_kv,
                                              int dtype) {
  if (tokens == 0 || seqs == 0) return 0;
  if (tokens < 0 || seqs < 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || dim <= 0 || max_q < 0 || max_kv < 0) return -1;
  const int group = heads / kv_heads;
  const long a = pg_ws_bytes(pg_plan(tokens, seqs, kv_heads, group, max_q, max_kv, false), tokens * heads, dim);
  const long b = pg_ws_bytes(pg_plan(tokens, seqs, kv_heads, group, max_q, max_kv, true), tokens * heads, dim);
  return a > b ? a : b;
}

template <typename T, int D, int NW>
static int pg_launch_tiles(const PgArgs<T>& a, long blocks, hipStream_t st) {
  constexpr int LDS = 4 * (D * sizeof(T) <= 256 ? 64 : 32) * D * sizeof(T);
  auto kern = paged_tile_kernel<T, D, NW>;
  if (LDS > 49152) {
    static focr_dev_flags done;
    if (focr_dev_first(done)) {
      if (hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, LDS) != hipSuccess) return FOCR_EHIP;
      focr_dev_mark(done);
    }
  }
  hipLaunchKernelGGL(kern, dim3((unsigned)blocks), dim3(64 * NW), LDS, st, a);
  return FOCR_OK;
}

template <typename T, int D>
static int pg_run(PgArgs<T> a, long ws_bytes, hipStream_t st) {
  const PagedShape& c = a.c;
  PgPlan p = pg_plan(c.tokens, c.seqs, a.kv_heads, a.group, a.max_q, c.max_kv, c.q_start != nullptr);
  constexpr bool WIDE = D * sizeof(T) <= 512;          // fp32 x 256: a wave's queries and sums need the registers of two
  if (!WIDE) p.tile_waves = 4;
  a.nsplit = p.nsplit;
  a.chunk = p.chunk;
  a.tile_chunk = p.tile_chunk;
  a.thin_rows = p.thin_rows;
  const long rows = c.tokens * a.heads, need = pg_ws_bytes(p, rows, D);
  if (need) {
    if (!a.part || ws_bytes < need) return FOCR_EINVAL;
    a.ml = (float2*)(a.part + need / ((D + 2) * 4) * D);
  }
  const long thin = (long)p.nsplit * a.kv_heads * c.seqs;
  const long per_head = paged_tiles(c.tokens, c.seqs, a.group, 32 * p.tile_waves), tiles = per_head * a.kv_heads * p.tsplit;
  // a launch has at most 2^32 threads in a direction
  if (thin >> 24 || tiles >> 23 || rows > INT32_MAX - 4096 || (need && rows >> 26)) return FOCR_EUNSUPPORTED;
  a.tiles = (int)per_head;
  if ((long)a.max_q * a.group > 32) {
    int rc;
    if constexpr (WIDE) rc = p.tile_waves == 8 ? pg_launch_tiles<T, D, 8>(a, tiles, st) : pg_launch_tiles<T, D, 4>(a, tiles, st);
    else rc = pg_launch_tiles<T, D, 4>(a, tiles, st);
    if (rc) return rc;
  }
  if (p.thin_rows > 16) hipLaunchKernelGGL((paged_thin_kernel<T, D, 2>), dim3((unsigned)thin), dim3(256), 0, st, a);
  else if (p.thin_rows) hipLaunchKernelGGL((paged_thin_kernel<T, D, 1>), dim3((unsigned)thin), dim3(256), 0, st, a);
  if (need) {
    if ((p.nsplit > 16 || p.tsplit > 16) && rows >> 24 == 0) hipLaunchKernelGGL((paged_join_kernel<T, D, 4>), dim3((unsigned)rows), dim3(256), 0, st, a);
    else hipLaunchKernelGGL((paged_join_kernel<T, D, 1>), dim3(cdiv(rows, 4)), dim3(256), 0, st, a);
  }
  return FOCR_OK;
}

extern "C" int focr_paged_attention_fwd(const void* q, long ldt, long ldh, const void* k_pages, const void* v_pages,
                                        const int* table, const int* kv_lens, const int* q_start, void* o, long ldto, long ldho,
                                        void* ws, long ws_bytes, long tokens, int seqs, int heads, int kv_heads, int dim,
                                        int page, int table_ld, long num_pages, int max_q, int max_kv, float scale, int causal,
                                        int dtype, void* stream) {
  PG_CHECK_COMMON();
  FOCR_CHECK_ARG(q && o, "null pointer");
  FOCR_CHECK_ARG(kv_heads > 0 && heads > 0 && heads % kv_heads == 0, "heads must be a multiple of kv_heads");
  FOCR_CHECK_ARG(max_q >= 0 && max_kv >= 0 && max_kv <= INT32_MAX - 16384, "max_q / max_kv out of range");
  FOCR_CHECK_ARG(pg_aligned(ws), "workspace must be 16-byte aligned");
  FOCR_CHECK_ARG(scale > 0.f && scale < INFINITY, "scale must be positive and finite");
  FOCR_CHECK_ARG(q_start || tokens / seqs <= max_q, "max_q is below tokens / seqs");
  PagedShape c;
  FOCR_CHECK_ARG(pg_shape(c, table, kv_lens, q_start, tokens, seqs, page, table_ld, num_pages, max_kv),
                 "page must be a power of two from 8 to 1024");
  const long es = pg_esize(dtype), cache = num_pages * kv_heads * page * dim * es;
  const long qb = ((tokens - 1) * ldt + (heads - 1) * ldh + dim) * es, ob = ((tokens - 1) * ldto + (heads - 1) * ldho + dim) * es;
  FOCR_CHECK_ARG(!focr_overlap(o, ob, q, qb) && !focr_overlap(o, ob, k_pages, cache) && !focr_overlap(o, ob, v_pages, cache),
                 "the output shares memory with q or the cache");
  int rc;
  const bool wq = pg_aligned(q) && (((ldt | ldh) * es) & 15) == 0;
  const bool wo = pg_aligned(o) && (((ldto | ldho) * es) & 15) == 0;
#define PG_RUN(T, DD)                                                                                                       \
  rc = pg_run<T, DD>(PgArgs<T>{(const T*)q, ldt, ldh, (const T*)k_pages, (const T*)v_pages, c, (T*)o, ldto, ldho, (float*)ws, \
                               nullptr, max_q, heads, kv_heads, heads / kv_heads, 1, 0, 0, 0, causal ? 1 : 0, 0, wq, wo,             \
                               scale * 1.4426950408889634f}, ws_bytes, (hipStream_t)stream)
#define PG_RUN_D(T)                    \
  if (dim == 64) PG_RUN(T, 64);        \
  else if (dim == 128) PG_RUN(T, 128); \
  else PG_RUN(T, 256)
  if (dtype == FOCR_DT_F32) { PG_RUN_D(float); }
  else if (dtype == FOCR_DT_BF16) { PG_RUN_D(bf16_t); }
  else { PG_RUN_D(f16_t); }
  FOCR_CHECK_ARG(rc != FOCR_EINVAL, "workspace missing or too small (focr_paged_attention_ws_bytes)");
  if (rc == FOCR_EHIP) {
    focr_set_error("%s: hipFuncSetAttribute failed", __func__);
    return rc;
  }
  if (rc == FOCR_EUNSUPPORTED) {
    focr_set_error("%s: too many sequences, heads and splits for one launch", __func__);
    return rc;
  }
  FOCR_LAUNCH_CHECK();
  return FOCR_OK;
}
