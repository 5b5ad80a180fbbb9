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
//
// One pass over the logits: a wave takes a segment of a row, 2048 values at a time in registers, and keeps
//   * per lane the running maximum and the sum of exp(x - maximum) in 64 bits.  The exponential is 13 full-rate fp64 operations
//     (a multiple of ln 2 taken off by a rounding addition, a polynomial of degree 7 on the rest: 6e-11), about what the
//     loads of 16-bit logits cost in time; a hardware exp2 in fp32 would be off by 1e-7, as far apart as neighbours can be;
//   * nothing else: afterwards the n-th largest of the lanes' maxima is a lower bound of the n-th best, only the few lanes whose
//     maximum reaches it hold candidates, and their values are read again, 16 bytes a lane, all at once.  Little more than n pass;
//     they are appended to a buffer by ballot, as 64-bit keys (the value's bits in an order that compares as integers, then the
//     complement of the index), and put in order at the end.  (A bound that grows with the chunks, candidates taken from
//     the registers: 45 us at 64 x 8 x 50001 where this takes 36.)  Rows of nearly one value -- a vocabulary masked to a few
//     tokens -- have all lanes read again, in order: 62 us at that size (fp32 79, where other rows take 38).
// Segments start at fixed indices and lanes take fixed indices of them whatever the row's alignment, so equal rows have
// equal sums.  A second pass over K x segments lists of n joins them (in the same block where a batch entry is small).
// Measured (64 entries x 8 beams x 50001, bf16, 51 MB): scan 27 us -- 12 for the loads alone, 12 more for the exponentials, the rest
// for the candidates -- and 7 us for the join; 33 us a call.
#define BS_CHUNK 2048
#define BS_MAX 64                     // beams, and candidates asked for
#define BS_WAVES 16                   // of the one-launch form
#define BS_BUF 256                    // keys a wave gathers: more than twice BS_MAX
typedef unsigned long long u64_t;
typedef __attribute__((ext_vector_type(4))) uint32_t bs_u32x4;
typedef __attribute__((ext_vector_type(4), aligned(2))) uint32_t bs_u32x4_any;      // 16 bytes at any element's address

struct BsStat {                       // of a segment
  double sum;                         // of exp(x - max)
  float max;                          // NaN: the segment holds one
};

__device__ __forceinline__ uint32_t bs_order(float x) {           // -inf < .. < +inf as integers; both zeros alike, NaN as -inf
  const uint32_t b = __float_as_uint(x != x ? -INFINITY : x + 0.f);
  return b >> 31 ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float bs_value(u64_t key) {
  const uint32_t o = (uint32_t)(key >> 32);
  return __uint_as_float(o >> 31 ? o & 0x7fffffffu : ~o);
}
__device__ __forceinline__ int bs_index(u64_t key) { return (int)~(uint32_t)key; }
__device__ __forceinline__ u64_t bs_key(float x, int v) { return (u64_t)bs_order(x) << 32 | (uint32_t)~v; }

__device__ __forceinline__ double bs_exp(double t) {              // t <= 0; exp(-700) stands for everything below
  t = fmax(t, -700.0);
  const double u = fma(t, 1.4426950408889634, 6755399441055744.0);           // 1.5 * 2^52: rounds to an integer, kept in the low word
  const double r = fma(u - 6755399441055744.0, -0.6931471805599453, t);
  double p = 0.00019907582591804609;                              // interpolates exp at the Chebyshev nodes of |r| <= ln 2 / 2
  p = fma(p, r, 0.0013948590286876341);
  p = fma(p, r, 0.008333283518767049);
  p = fma(p, r, 0.04166621813971032);
  p = fma(p, r, 0.16666666786380446);
  p = fma(p, r, 0.5000000107793876);
  p = fma(p, r, 0.9999999999955055);
  p = fma(p, r, 0.9999999999595294);
  return __hiloint2double(__double2hiint(p) + (__double2loint(u) << 20), __double2loint(p));
}
// the largest value of the wave, in every lane: lane crossings inside the vector unit
__device__ __forceinline__ float bs_wave_max(float x) {
#define BS_STEP(ctrl) x = fmaxf(x, __int_as_float(__builtin_amdgcn_update_dpp((int)0xff800000, __float_as_int(x), ctrl, 0xf, 0xf, false)))
  BS_STEP(0x111);
  BS_STEP(0x112);
  BS_STEP(0x114);
  BS_STEP(0x118);
  BS_STEP(0x142);
  BS_STEP(0x143);
#undef BS_STEP
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), 63));
}

__device__ __forceinline__ u64_t bs_lane(u64_t x, int l) {
  return (u64_t)(uint32_t)__builtin_amdgcn_readlane((int)(x >> 32), l) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)x, l);
}
// key (the same in all lanes) into the sorted list across the lanes; what falls off its end is lost
__device__ __forceinline__ void bs_insert(u64_t& list, u64_t key, int lane) {
  const int at = __popcll(__ballot(list > key));
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(list >> 32), 0x138, 0xf, 0xf, false);      // from the lane below
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)list, 0x138, 0xf, 0xf, false);
  list = lane < at ? list : lane == at ? key : (u64_t)hi << 32 | lo;
}

// The n best of the buffer's cnt keys to out[0 .. n) in order (0 where there are fewer): every key finds its place by counting
// the ones above it
__device__ __forceinline__ void bs_trim(const u64_t* buf, int cnt, int n, int lane, u64_t* out) {
  if (lane >= cnt && lane < n) out[lane] = 0;
  constexpr int R = BS_BUF / 64;
  u64_t mine[R];
  int at[R] = {};
#pragma unroll
  for (int i = 0; i < R; ++i) mine[i] = i * 64 + lane < cnt ? buf[i * 64 + lane] : 0;
#pragma unroll
  for (int j = 0; j < R; ++j) {
    const int m = cnt - j * 64 < 64 ? cnt - j * 64 : 64;
    if (cnt <= 64) {
      for (int e = 0; e < m; ++e) at[0] += bs_lane(mine[j], e) > mine[0];
    } else {
      for (int e = 0; e < m; ++e) {
        const u64_t key = bs_lane(mine[j], e);
#pragma unroll
        for (int i = 0; i < R; ++i) at[i] += key > mine[i];
      }
    }
  }
#pragma unroll
  for (int i = 0; i < R; ++i)
    if (i * 64 + lane < cnt && at[i] < n) out[at[i]] = mine[i];
  __builtin_amdgcn_wave_barrier();
}

template <typename T, int L>          // L loads of 16 bytes a lane make a chunk
__device__ __forceinline__ void bs_scan(const T* row, int v0, int v1, int n, int lane, u64_t* buf, u64_t* best, BsStat& stat) {
  constexpr int E = 16 / sizeof(T), CHUNK = L * 64 * E;
  float m = -INFINITY, thr = -INFINITY, x[L * E];
  double sum = 0.0;
  bool nan = false, ahead = false;
  bs_u32x4 w[L];
  // 16 bytes of a row from `at` on; behind the row's end the last 16 of it, of which a lane takes what is its own
  auto from = [&](int at) { return at + E <= v1 ? at : v1 - E; };
  auto load = [&](int base) {
#pragma unroll
    for (int j = 0; j < L; ++j) w[j] = *(const bs_u32x4_any*)(row + from(base + (j * 64 + lane) * E));
  };
  for (int base = v0; base < v1; base += CHUNK) {
    if (v1 >= E) {
      if (!ahead) load(base);
#pragma unroll
      for (int i = 0; i < L * E; ++i) {
        if constexpr (sizeof(T) == 4) x[i] = __uint_as_float(w[i / E][i % E]);
        else x[i] = (float)__builtin_bit_cast(T, (uint16_t)(w[i / E][i % E / 2] >> (16 * (i & 1))));
        nan |= x[i] != x[i];
      }
      if (base + CHUNK > v1) {
#pragma unroll
        for (int i = 0; i < L * E; ++i) {
          const int at = base + (i / E * 64 + lane) * E;
          if (from(at) + i % E < at) x[i] = NAN;                  // another lane's: passes no comparison, adds nothing
        }
      }
    } else {                                                      // a row of less than 16 bytes: in lane 0
#pragma unroll
      for (int i = 0; i < L * E; ++i) {
        x[i] = NAN;
        if (i < E) {
          const float y = (float)row[i < v1 ? i : v1 - 1];
          nan |= y != y;
          if (i < v1 && lane == 0) x[i] = y;
        }
      }
    }
    ahead = base + CHUNK < v1;
    if (ahead) load(base + CHUNK);                                // under this chunk's arithmetic
    float cm = -INFINITY;
#pragma unroll
    for (int i = 0; i < L * E; ++i) cm = fmaxf(cm, x[i]);
    if (cm > m) {
      sum *= bs_exp((double)m - (double)cm);                      // (-inf before the first values: the sum is 0)
      m = cm;
    }
    const double ref = m == -INFINITY ? 0.0 : (double)m;
#pragma unroll
    for (int i = 0; i < L * E; ++i) {
      sum += bs_exp((double)x[i] - ref);                          // (-inf: 1e-304, nothing beside the maximum's 1)
      if (i % 4 == 3) __builtin_amdgcn_sched_barrier(0);          // four chains at a time fill the pipe; more only take registers
    }
  }

  if (L > 1 || v1 - v0 > 256) {                                   // the n-th largest of the lanes' maxima: values that are there
    if (n <= 16) {
      float y = m;
      for (int r = 0; r < n; ++r) {
        thr = bs_wave_max(y);
        if (lane == __builtin_ctzll(__ballot(y == thr) | 1ull << 63)) y = -INFINITY;
      }
    } else {
      int rank = 0;
#pragma unroll 8
      for (int j = 0; j < 64; ++j) {
        const float y = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(m), j));
        rank += y > m || (y == m && j < lane);
      }
      thr = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(m), __builtin_ctzll(__ballot(rank == n - 1) | 1ull << 63)));
    }
  }
  // Candidates to the buffer, a value a lane at a time.  Where they could run over (many equal values), the buffer goes back to
  // its n best first and takes what is above the last of them
  int cnt = 0, last = INT32_MAX;
  auto put = [&](bool in, u64_t key) {
    const u64_t pass = __ballot(in);
    if (in) buf[cnt + __builtin_amdgcn_mbcnt_hi((uint32_t)(pass >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)pass, 0))] = key;
    cnt += __popcll(pass);
  };
  auto take = [&](float (&y)[E], int (&v)[E]) {
    if (last == INT32_MAX) {                                      // the buffer was not cut yet: the bound alone counts
      int more = 0;
#pragma unroll
      for (int j = 0; j < E; ++j) more += __popcll(__ballot(y[j] >= thr));
      if (cnt + more <= BS_BUF) {
#pragma unroll
        for (int j = 0; j < E; ++j)
          if (__ballot(y[j] >= thr)) put(y[j] >= thr, bs_key(y[j], v[j]));
        return;
      }
    }
    const auto fits = [&](float y, int v) { return y > thr || (y == thr && v < last); };
    bool any = false;
#pragma unroll
    for (int j = 0; j < E; ++j) any |= fits(y[j], v[j]);
    if (!__ballot(any)) return;
#pragma unroll 1
    for (int g = 0; g < E; ++g) {
      if (cnt > n + 64) {
        __builtin_amdgcn_wave_barrier();
        bs_trim(buf, cnt, n, lane, best);
        const u64_t list = lane < n ? best[lane] : 0;
        if (lane < n) buf[lane] = list;
        cnt = n;
        thr = bs_value(bs_lane(list, n - 1));
        last = bs_index(bs_lane(list, n - 1));
      }
      put(fits(y[0], v[0]), bs_key(y[0], v[0]));
#pragma unroll
      for (int j = 1; j < E; ++j) y[j - 1] = y[j], v[j - 1] = v[j];
    }
  };
  if (L == 1 || v1 < E) {                                         // a single chunk: the values are still there
    float y[E];
    int v[E];
#pragma unroll
    for (int i = 0; i < E; ++i) y[i] = x[i], v[i] = v1 >= E ? from(v0 + lane * E) + i : i;
    take(y, v);
  } else {
    // only the lanes whose maximum reaches the threshold hold any.  Their values are read again by the whole wave, 16 bytes a lane
    const bool has = m >= thr && lane * E < v1 - v0;
    const u64_t some = __ballot(has);
    const int rank = __builtin_amdgcn_mbcnt_hi((uint32_t)(some >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)some, 0));
    const int lanes = __popcll(some), pieces = (v1 - v0 + 64 * E - 1) / (64 * E), items = lanes * pieces;
    const int who = __builtin_amdgcn_ds_permute(4 * (has ? rank : lanes + lane - rank), lane);      // those lanes first
    for (int i0 = 0; i0 < items; i0 += 4 * 64) {
      bs_u32x4 z[4];
      int at[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {                               // four loads on their way together
        const int i = i0 + j * 64 + lane, q = i / lanes, l = __builtin_amdgcn_ds_bpermute(4 * (i - q * lanes), who);
        at[j] = i < items ? v0 + (q * 64 + l) * E : v1;
        z[j] = *(const bs_u32x4_any*)(row + from(at[j]));
      }
#pragma unroll 1
      for (int j = 0; j < 4 && i0 + j * 64 < items; ++j) {
        float y[E];
        int v[E];
#pragma unroll
        for (int i = 0; i < E; ++i) {
          if constexpr (sizeof(T) == 4) y[i] = __uint_as_float(z[0][i]);
          else y[i] = (float)__builtin_bit_cast(T, (uint16_t)(z[0][i / 2] >> (16 * (i & 1))));
          v[i] = from(at[0]) + i;
          if (v[i] < at[0]) y[i] = NAN;
        }
        take(y, v);
#pragma unroll
        for (int k = 1; k < 4; ++k) z[k - 1] = z[k], at[k - 1] = at[k];
      }
    }
  }
  __builtin_amdgcn_wave_barrier();
  bs_trim(buf, cnt, n, lane, best);
  const float mx = bs_wave_max(m);
  sum = m == -INFINITY ? 0.0 : sum * bs_exp((double)m - (double)mx);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
  stat.max = __ballot(nan) ? NAN : mx;
  stat.sum = sum;
}

struct BsArgs {
  const void* logits;
  long ldb, ldk;
  const float* scores;
  const uint8_t* fin;
  float* out_scores;
  int* out_parents;
  long long* out_tokens;
  uint8_t* out_fin;
  u64_t* lists;                       // [batch][beams][parts][n]
  BsStat* stats;                      // [batch][beams][parts]
  int beams, vocab, n, eos, parts, seg;
};

__device__ __forceinline__ bool bs_before(double ca, int ia, double cb, int ib) { return ca > cb || (ca == cb && ia < ib); }

struct BsBeam {
  float score;
  bool done;
};
__device__ __forceinline__ BsBeam bs_beam(const BsArgs& a, int b, int k) {
  const int i = b * a.beams + (k < a.beams ? k : 0);
  return {a.scores[i], a.fin && a.fin[i]};
}

// Joins the lists of a batch entry (waves: of the block; lists / stats of this entry; own: bs_beam of the wave's first beam).
// rc / rv / rp [beams][n]: the rows' candidates and their places
__device__ __forceinline__ void bs_join(const BsArgs& a, int b, const u64_t* lists, const BsStat* stats, double* rc, int* rv,
                                        int* rp, int waves, BsBeam own) {
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), n = a.n;
  const int have = n < a.vocab ? n : a.vocab;                     // candidates of a row
  for (int k = wave; k < a.beams; k += waves) {
    const BsBeam beam = k == wave ? own : bs_beam(a, b, k);
    u64_t list = lane < n ? lists[(long)k * a.parts * n + lane] : 0;
    BsStat first = {0.0, -INFINITY};                              // all loads before the work on any
    if (lane < a.parts) first = stats[k * a.parts + lane];
    for (int p0 = 1; p0 < a.parts; p0 += 8) {                     // eight loads at a time, then their turn
      u64_t other[8];
#pragma unroll
      for (int j = 0; j < 8; ++j)
        other[j] = lane < n && p0 + j < a.parts ? lists[((long)k * a.parts + p0 + j) * n + lane] : 0;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        for (int i = 0; i < n; ++i) {
          const u64_t key = bs_lane(other[j], i);
          if (key <= bs_lane(list, n - 1)) break;
          bs_insert(list, key, lane);
        }
    }
    float m = first.max;
    bool nan = m != m;
    for (int p = 64 + lane; p < a.parts; p += 64) {
      const float x = stats[k * a.parts + p].max;
      nan |= x != x;
      m = fmaxf(m, x);
    }
    m = bs_wave_max(m);
    double sum = first.max > -INFINITY ? first.sum * bs_exp((double)first.max - (double)m) : 0.0;
    for (int p = 64 + lane; p < a.parts; p += 64) {
      const BsStat st = stats[k * a.parts + p];
      if (st.max > -INFINITY) sum += st.sum * bs_exp((double)st.max - (double)m);
    }
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
    const float s = beam.score;
    const bool done = beam.done;
    const bool live = isfinite(s) && (done || (!__ballot(nan) && isfinite(m)));
    double c = -INFINITY;
    int v = lane;
    if (live && done) {                                           // (eos, s), then the others as they come
      v = lane == 0 ? a.eos : lane <= a.eos ? lane - 1 : lane;
      if (lane == 0) c = (double)s;
    } else if (live) {
      v = bs_index(list);
      c = (double)s - ((double)m + log(sum)) + (double)bs_value(list);
    }
    // in order of (candidate, index): 64 bits may round different logits to one candidate
    int at = 0;
    for (int j = 0; j < have; ++j) {
      const double cj = __shfl(c, j, 64);
      const int vj = __shfl(v, j, 64);
      at += j != lane && bs_before(cj, vj, c, v);
    }
    if (lane < have) {
      rc[k * n + at] = c;
      rv[k * n + at] = v;
      rp[k * n + at] = done ? at | 1 << 30 : at;
    }
  }
  __syncthreads();
  // a candidate's place: its place in its own row plus, by bisection, how many of every other row come before it
  const int all = a.beams * have;
  for (int x = tid; x < all * a.beams; x += waves * 64) {
    const int r = x / all, y = x - r * all, k = y / have, i = y - k * have;
    if (r == k) continue;
    const double c = rc[k * n + i];
    int lo = 0, hi = have;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      const double cm = rc[r * n + mid];
      if (cm > c || (cm == c && r < k)) lo = mid + 1;
      else hi = mid;
    }
    atomicAdd(&rp[k * n + i], lo);                                // whole numbers: the same in any order
  }
  __syncthreads();
  for (int x = tid; x < all; x += waves * 64) {
    const int k = x / have, i = k * n + x - k * have, at = rp[i] & (1 << 30) - 1, v = rv[i];
    if (at >= n) continue;
    a.out_scores[b * n + at] = (float)rc[i];
    a.out_parents[b * n + at] = k;
    a.out_tokens[b * n + at] = v;
    a.out_fin[b * n + at] = rp[i] >> 30 || v == a.eos;
  }
}

// a whole batch entry in a block: wave (beam, segment)
template <typename T, int L>
__global__ __launch_bounds__(64 * BS_WAVES) void beam_select_kernel(BsArgs a) {
  __shared__ u64_t buf[BS_WAVES * BS_BUF], lists[BS_WAVES * BS_MAX];
  __shared__ BsStat stats[BS_WAVES];
  __shared__ double rc[BS_WAVES * BS_MAX];
  __shared__ int rv[BS_WAVES * BS_MAX], rp[BS_WAVES * BS_MAX];
  const int b = blockIdx.x, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int k = wave / a.parts, p = wave - k * a.parts;
  const BsBeam own = bs_beam(a, b, wave);
  BsStat st;
  const int v0 = p * a.seg, v1 = v0 + a.seg < a.vocab ? v0 + a.seg : a.vocab;
  bs_scan<T, L>((const T*)a.logits + b * a.ldb + k * a.ldk, v0, v1, a.n, lane, buf + wave * BS_BUF, lists + wave * a.n, st);
  if (lane == 0) stats[wave] = st;
  __syncthreads();
  bs_join(a, b, lists, stats, rc, rv, rp, a.beams * a.parts, own);
}

// the two-launch form
template <typename T>
__global__ __launch_bounds__(256, 4) void beam_scan_kernel(BsArgs a, int waves) {
  __shared__ u64_t buf[4 * BS_BUF], best[4 * BS_MAX];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), w = blockIdx.x * 4 + wave;
  if (w >= waves) return;
  const int p = w % a.parts, row = w / a.parts, b = row / a.beams, k = row - b * a.beams;
  BsStat st;
  const int v0 = p * a.seg, v1 = v0 + a.seg < a.vocab ? v0 + a.seg : a.vocab;
  bs_scan<T, BS_CHUNK * sizeof(T) / 1024>((const T*)a.logits + b * a.ldb + k * a.ldk, v0, v1, a.n, lane, buf + wave * BS_BUF,
                                          best + wave * BS_MAX, st);
  if (lane < a.n) a.lists[(long)w * a.n + lane] = best[wave * BS_MAX + lane];
  if (lane == 0) a.stats[w] = st;
}
__global__ __launch_bounds__(64 * BS_WAVES) void beam_join_kernel(BsArgs a, int waves) {
  extern __shared__ double bs_rc[];                               // [beams][n], then the indices, then the places
  const long rows = (long)blockIdx.x * a.beams * a.parts;
  int* rv = (int*)(bs_rc + a.beams * a.n);
  bs_join(a, blockIdx.x, a.lists + rows * a.n, a.stats + rows, bs_rc, rv, rv + a.beams * a.n, waves,
          bs_beam(a, blockIdx.x, __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)));
}

// One launch with a block per batch entry while an entry has at most 16 K logits; else the rows are cut into segments of whole
// chunks, about 2048 waves in all (64 x 8 x 50001 bf16: 33 us, twice as many 36.5), and joined by a second launch.  A call of 64
// entries x 5 beams, fp32, in one / two launches: 2000 classes 10.9 / 14.7 us, 3270 (16 K logits) 13.4 / 14.6, 4500 15.3 / 14.4, 6625
// 16.9 / 14.6; of 1 and 16 entries the same within 1 us, of 128 at 6625 both 17.5.
struct BsPlan {
  bool one;
  int parts, seg;
};
static BsPlan bs_plan(int batch, int beams, int vocab) {
  const int chunks = (vocab + BS_CHUNK - 1) / BS_CHUNK;
  BsPlan p;
  p.one = beams <= BS_WAVES && (long)beams * vocab <= 16384;
  const long want = p.one ? BS_WAVES / beams : 2048 / ((long)batch * beams);
  const int per = want < 1 ? chunks : (int)((chunks + want - 1) / want);
  p.seg = per * BS_CHUNK;
  p.parts = (chunks + per - 1) / per;
  return p;
}

extern "C" long focr_beam_select_ws_bytes(int batch, int beams, int vocab, int n, int dtype) {
  if (batch <= 0 || beams <= 0 || vocab <= 0 || n <= 0) return 0;
  const BsPlan p = bs_plan(batch, beams, vocab);
  return p.one ? 0 : (long)batch * beams * p.parts * (n * (long)sizeof(u64_t) + (long)sizeof(BsStat));
}

extern "C" int focr_beam_select(const void* logits, long ldb, long ldk, const float* scores, const uint8_t* finished,
                                float* out_scores, int* out_parents, long long* out_tokens, uint8_t* out_finished, void* ws,
                                long ws_bytes, int batch, int beams, int vocab, int n, int eos, int dtype, void* stream) {
  FOCR_CHECK_ARG(dtype == FOCR_DT_F32 || dtype == FOCR_DT_BF16 || dtype == FOCR_DT_F16, "dtype must be fp32, bf16 or fp16");
  FOCR_CHECK_ARG(batch >= 0 && beams > 0 && beams <= BS_MAX && vocab > 0 && vocab < INT32_MAX - 2 * BS_CHUNK,
                 "beams must be 1 to 64, vocab positive");
  FOCR_CHECK_ARG(n > 0 && n <= BS_MAX && n <= (long)beams * vocab, "n must be 1 to 64 and at most beams * vocab");
  FOCR_CHECK_ARG(!finished || (eos >= 0 && eos < vocab), "finished beams need an eos inside the vocabulary");
  if (batch == 0) return FOCR_OK;
  FOCR_CHECK_ARG(logits && scores && out_scores && out_parents && out_tokens && out_finished, "null pointer");
  const BsPlan p = bs_plan(batch, beams, vocab);
  const long rows = (long)batch * beams * p.parts;
  FOCR_CHECK_ARG(rows >> 26 == 0 && batch >> 22 == 0, "too many rows for one launch");
  FOCR_CHECK_ARG(p.one || (ws && ((uintptr_t)ws & 7) == 0 && ws_bytes >= focr_beam_select_ws_bytes(batch, beams, vocab, n, dtype)),
                 "workspace missing or too small (focr_beam_select_ws_bytes)");
  BsArgs a = {logits, ldb, ldk, scores, finished, out_scores, out_parents, out_tokens, out_finished, (u64_t*)ws,
              p.one ? nullptr : (BsStat*)((u64_t*)ws + rows * n), beams, vocab, n, eos, p.parts, p.seg};
  const hipStream_t st = (hipStream_t)stream;
  if (p.one) {
    // a handful of classes: one load a lane, an eighth of the instructions to fetch and run through
#define BS_KERN(T) (vocab <= 1024 / (int)sizeof(T) ? beam_select_kernel<T, 1> : beam_select_kernel<T, BS_CHUNK * sizeof(T) / 1024>)
    auto kern = dtype == FOCR_DT_F32 ? BS_KERN(float) : dtype == FOCR_DT_BF16 ? BS_KERN(__bf16) : BS_KERN(_Float16);
    hipLaunchKernelGGL(kern, dim3(batch), dim3(64 * beams * p.parts), 0, st, a);
  } else {
    auto kern = dtype == FOCR_DT_F32 ? beam_scan_kernel<float> : dtype == FOCR_DT_BF16 ? beam_scan_kernel<__bf16> : beam_scan_kernel<_Float16>;
    hipLaunchKernelGGL(kern, dim3(cdiv(rows, 4)), dim3(256), 0, st, a, (int)rows);
    FOCR_LAUNCH_CHECK();
    const int waves = beams < BS_WAVES ? beams : BS_WAVES;
    hipLaunchKernelGGL(beam_join_kernel, dim3(batch), dim3(64 * waves), beams * n * 16, st, a, waves);
  }
  FOCR_LAUNCH_CHECK();
  return FOCR_OK;
}

// ======================================================================================================================
// Reordering.  The beams of a group have the same length L; beam j goes on from beam p = parents[j].  Full pages are never
// written again, so j takes p's table entries for them.  The last, partial page (L % page tokens) will be written by every
// beam: a j != p gets its own copy, in its spare page, and the page it held before becomes its spare.  So a beam moves at most
// page - 1 tokens however long the sequence, and no page is allocated or freed.  Bound by the bytes moved: 64 x 8 beams, 4 layers of
// 8 x 128 bf16, pages of 64: 87 us for 209 MB written and as many read, in runs of 8 KB (4.8 TB/s; a large copy: 4.9), a call
// 94 .. 102 us.
// ======================================================================================================================
#define BR_MAX_TENSORS 64
#define BR_PIECE 1024                 // 16-byte units a block moves (512 .. 2048: 97 .. 110 us)
struct BrPages {
  char* p[BR_MAX_TENSORS];
};

__device__ __forceinline__ int br_parent(const int* parents, int slot, int beams) {
  const int p = parents[slot];
  return p >= 0 && p < beams ? slot / beams * beams + p : slot;          // no such beam: the slot goes on from itself
}

// grid (BR_PIECE units of a page, slot, tensor).  Where the tables that go out are not the ones that come in (table_out), the
// blocks behind the last tensor write them in the same launch
__global__ __launch_bounds__(256) void beam_copy_pages_kernel(BrPages pages, int tensors, const int* __restrict__ parents,
                                                              const int* __restrict__ table, const int* __restrict__ lens,
                                                              const int* __restrict__ spare, int* __restrict__ table_out,
                                                              int* __restrict__ spare_out, int beams, int heads, int row_units,
                                                              int page_shift, int table_ld, long num_pages) {
  const int slot = blockIdx.y, src_slot = br_parent(parents, slot, beams);
  const int len = lens[slot / beams * beams], full = len >> page_shift, rest = len & ((1 << page_shift) - 1);
  if ((int)blockIdx.z == tensors) {
    const bool ok = len >= 0 && (full < table_ld || (full == table_ld && rest == 0)), move = ok && rest && src_slot != slot;
    const int *own = table + (long)slot * table_ld, *src = table + (long)src_slot * table_ld;
    for (int col = blockIdx.x * 256 + threadIdx.x; col < table_ld; col += gridDim.x * 256)
      table_out[(long)slot * table_ld + col] = ok && col < full ? src[col] : move && col == full ? spare[slot] : own[col];
    if (blockIdx.x == 0 && threadIdx.x == 0) spare_out[slot] = move ? own[full] : spare[slot];
    return;
  }
  if (src_slot == slot || len < 0 || full >= table_ld || rest == 0) return;
  const int from = table[(long)src_slot * table_ld + full], to = spare[slot];
  if (from < 0 || from >= num_pages || to < 0 || to >= num_pages) return;
  const int run = rest * row_units, total = heads * run;                 // 16-byte units
  const long head_units = (long)row_units << page_shift;
  const long s = (long)from * heads * head_units, d = (long)to * heads * head_units;
  // head of a unit: x / run by one multiplication where that is exact (m = ceil(2^32 / run): x (m run - 2^32) < x run < 2^32)
  const uint32_t magic = 0xffffffffu / (uint32_t)run + 1;
  const bool quick = (uint64_t)total * (uint32_t)run < 1ull << 32 && run > 1;
  if ((int)blockIdx.x * BR_PIECE >= total) return;
  const int x0 = blockIdx.x * BR_PIECE + threadIdx.x;
  long at[BR_PIECE / 256];
#pragma unroll
  for (int i = 0; i < BR_PIECE / 256; ++i) {
    const int x = x0 + i * 256 < total ? x0 + i * 256 : total - 1, h = quick ? (int)__umulhi((uint32_t)x, magic) : x / run;
    at[i] = h * head_units + (x - h * run);
  }
  bs_u32x4* p = (bs_u32x4*)pages.p[blockIdx.z];
  bs_u32x4 v[BR_PIECE / 256];
#pragma unroll
  for (int i = 0; i < BR_PIECE / 256; ++i) v[i] = p[s + at[i]];          // all on their way before the first store
#pragma unroll
  for (int i = 0; i < BR_PIECE / 256; ++i)
    if (x0 + i * 256 < total) p[d + at[i]] = v[i];
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
  const long slots = (long)groups * beams;
  const long tb = slots * table_ld * 4, sb = slots * 4;
  const bool t_apart = !focr_overlap(table_out, tb, table, tb), s_apart = !focr_overlap(spare_out, sb, spare, sb), apart = t_apart && s_apart;
  FOCR_CHECK_ARG((t_apart || table_out == table) && (s_apart || spare_out == spare) && !focr_overlap(table_out, tb, spare_out, sb) &&
                     !focr_overlap(table_out, tb, spare, sb) && !focr_overlap(spare_out, sb, table, tb) &&
                     !focr_overlap(table_out, tb, parents, sb) && !focr_overlap(spare_out, sb, parents, sb) &&
                     !focr_overlap(table_out, tb, kv_lens, sb) && !focr_overlap(spare_out, sb, kv_lens, sb),
                 "table_out / spare_out share memory with another argument (they may be table / spare themselves)");
  for (int i = 0; i < tensors; i += BR_MAX_TENSORS) {
    BrPages b = {};
    const int m = tensors - i < BR_MAX_TENSORS ? tensors - i : BR_MAX_TENSORS;
    for (int j = 0; j < m; ++j) b.p[j] = (char*)pages[i + j];
    const bool tables = apart && i + m == tensors;
    hipLaunchKernelGGL(beam_copy_pages_kernel, dim3(cdiv(page_bytes, 16 * BR_PIECE), slots, m + (tables ? 1 : 0)), dim3(256), 0,
                       (hipStream_t)stream, b, m, parents, table, kv_lens, spare, table_out, spare_out, beams, heads,
                       (int)(row_bytes / 16), shift, table_ld, num_pages);
    FOCR_LAUNCH_CHECK();
  }
  if (apart && tensors) return FOCR_OK;
  hipLaunchKernelGGL(beam_tables_kernel, dim3(cdiv(table_ld, 256), groups), dim3(256), beams * 1024, (hipStream_t)stream,
                     parents, table, kv_lens, spare, table_out, spare_out, beams, shift, table_ld);
  FOCR_LAUNCH_CHECK();
  return FOCR_OK;
}
