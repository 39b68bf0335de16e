// az_sample.hip -- drawing one action per row of scores: temperature, top-k, top-p, min-p, from given uniform numbers (gfx950).
//
//   legal i: scores that are neither masked, NaN nor -inf;  m = max s;  w_i = exp((s_i - m) / T)
//   order: s descending, equal scores by ascending index;   K1 = the first top_k of it
//   kept:  i in K1 whose mass of K1 before it is < top_p * mass(K1) (the first one always), and w_i >= min_p
//   drawn: the smallest index i with (kept mass up to and including i) > u * (kept mass)
//
// Masses are held as 64-bit integers in units of 2^-44 of the largest weight: integer sums do not depend on their order, so
// histograms may be built with atomics and the drawn index is the same on every run and for every launch shape.  A weight is
// rounded once, by at most 2^-45 of the largest; an f32 mass (2^-24) would move the border between neighbours of long rows.
// At most 2^19 scores per row keep the sum below 2^63.
//
// The kept set is a prefix of the order, so it is described by its last member (key, index), and no row is ever sorted.
//
//   n <= 1,024: a row is one wave's, in registers; the prefix's end is bisected over the score, counting with ballots
//   longer:     a row is one workgroup's, which walks it twice where it can (the second time it comes from the caches): the first
//               walk leaves the largest scores of 1,024 shares of the row; what nine sixteenths of these reach (or k of them, for the top k),
//               some 820 scores do where large ones lie anywhere; the second walk lists those in LDS and bounds the mass in f32.  If
//               the prefix ends within the list, the rest is done on it.  A longer prefix is found from a histogram linear in the
//               score and a list of the bin it ends in.
//
// Bound by instructions and, in long rows, by latencies: about ten instructions a score and walk, and 25 f64 operations an exponential where the
// kept scores are many.  Measured (long rows: scores of deviation 3):
//   16,384 x 225 f32, masks, top k 16, top p 0.9, min p:   37 us (20.6 k vector instructions a SIMD, 34 us at four cycles each; the 18.6 MB
//                                                          would take 3.7)
//   1 x 225 f32:                                           5.4 us, the latency of one wave's steps; the call 12 us
//   512 x 65,537 bf16, T 0.7, top p 0.9, min p:            93 us (67 MB, read twice: 1.4 TB/s; 22.1 k vector instructions a SIMD take 37 us of it, and two waves
//                                                          a SIMD do not cover the walks' loads and the list's steps between barriers)
//     T 1, top p 0.9:                                      250 us: the prefix has more than 1,024 members, the list overflows, and of six walks two
//                                                          take an f64 exponential of every score
//     T 0.8, top k 50, top p 0.95 / T 1, no cut:           48 / 80 us
//   1 x 131,072 bf16, T 0.8, top k 50, top p 0.95:         38 us on one CU: a row is not shared out, its sums and lists stay in LDS; T 1, top p 0.9: 196 us
#include "az_ops.hip.h"

namespace azsample {

using namespace azops;
typedef unsigned long long u64;

constexpr int MAX_N = 1 << 19, BINS = 2048, LIST = 1024;
constexpr uint32_t KEY_NONE = 0x007FFFFFu;  // the image of -inf: masked, NaN and -inf scores
constexpr uint32_t KEY_PINF = 0xFF800000u;
constexpr double UNIT = 17592186044416.0;  // 2^44

struct Args {
  const void *scores;
  const uint8_t *legal;
  const float *u, *t_rows, *p_rows, *mp_rows;
  const int32_t *k_rows;
  int32_t *actions;
  float *logp;
  int64_t stride, legal_stride;
  double t, p, mp;
  int32_t k, n;
};

__device__ __forceinline__ uint32_t key_of(float s) {
  if (!(s > -INFINITY)) return KEY_NONE;
  const uint32_t b = __float_as_uint(s + 0.0f);  // -0 and +0 are one score
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float score_of(uint32_t key) { return __uint_as_float((key & 0x80000000u) ? (key & 0x7FFFFFFFu) : ~key); }

// 2^44 exp((s - m) / T) rounded to an integer, of N scores side by side (they share the constants and fill each other's latencies);
// sc = log2(e) / T.  2^f on [-1/2, 1/2] by its Taylor polynomial of degree 12 (remainder below 2^-51); scores of +inf share the whole
// mass.
template <int N> __device__ __forceinline__ void weights(const uint32_t *key, double m, double sc, bool inf_row, u64 *w) {
  if (inf_row) {
#pragma unroll
    for (int j = 0; j < N; ++j) w[j] = key[j] == KEY_PINF ? (u64)UNIT : 0;
    return;
  }
  double f[N], r[N];
  int e[N];
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const double y = __builtin_fmax(((double)score_of(key[j]) - m) * sc, -100.0), k = rint(y);
    f[j] = (y - k) * 0.693147180559945309417;
    e[j] = (int)k + 44;
    r[j] = 1.0 / 479001600.0;
  }
  constexpr double C[12] = {1.0 / 39916800.0, 1.0 / 3628800.0, 1.0 / 362880.0, 1.0 / 40320.0, 1.0 / 5040.0, 1.0 / 720.0, 1.0 / 120.0, 1.0 / 24.0, 1.0 / 6.0, 0.5, 1.0, 1.0};
#pragma unroll
  for (int d = 0; d < 12; ++d) {
#pragma unroll
    for (int j = 0; j < N; ++j) r[j] = fma(r[j], f[j], C[d]);
  }
  // 2^52 + w: the integer stands in the low mantissa bits, rounded to nearest even (w <= 2^44)
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const u64 v = (u64)__double_as_longlong(ldexp(r[j], e[j]) + 4503599627370496.0) & 0xFFFFFFFFFFFFFull;
    w[j] = key[j] == KEY_NONE ? 0 : v;
  }
}
__device__ __forceinline__ u64 weight(uint32_t key, double m, double sc, bool inf_row) {
  u64 w;
  weights<1>(&key, m, sc, inf_row, &w);
  return w;
}

// Wave reductions by data-parallel moves (rows of 16 lanes, then across rows): no LDS round trips.  The result is in lane 63 of a scan.
template <int CTRL, int ROWS> __device__ __forceinline__ uint32_t moved(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, false);
}
template <int CTRL, int ROWS> __device__ __forceinline__ u64 moved(u64 v) {
  return ((u64)moved<CTRL, ROWS>((uint32_t)(v >> 32)) << 32) | moved<CTRL, ROWS>((uint32_t)v);
}
template <class N> __device__ __forceinline__ N wave_scan(N v) {  // inclusive sum over lanes
  v += moved<0x111, 0xF>(v);  // row_shr 1, 2, 4, 8
  v += moved<0x112, 0xF>(v);
  v += moved<0x114, 0xF>(v);
  v += moved<0x118, 0xF>(v);
  v += moved<0x142, 0xA>(v);  // row_bcast 15 into rows 1 and 3
  v += moved<0x143, 0xC>(v);  // row_bcast 31 into rows 2 and 3
  return v;
}
__device__ __forceinline__ u64 lane_of(u64 v, int lane) {
  return ((u64)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32) | (uint32_t)__builtin_amdgcn_readlane((int)v, lane);
}
__device__ __forceinline__ u64 wave_sum(u64 v) { return lane_of(wave_scan(v), 63); }
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
  auto up = [&](uint32_t x) { v = x > v ? x : v; };
  up(moved<0x111, 0xF>(v));
  up(moved<0x112, 0xF>(v));
  up(moved<0x114, 0xF>(v));
  up(moved<0x118, 0xF>(v));
  up(moved<0x142, 0xA>(v));
  up(moved<0x143, 0xC>(v));
  return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}

struct Setting {  // of one row
  double sc, p, least;
  int k;
  float u;
};
__device__ __forceinline__ Setting setting_of(const Args &a, int64_t r) {
  double t = a.t_rows ? (double)a.t_rows[r] : a.t;
  const double mp = a.mp_rows ? (double)a.mp_rows[r] : a.mp;
  Setting s;
  s.p = a.p_rows ? (double)a.p_rows[r] : a.p;
  s.k = a.k_rows ? a.k_rows[r] : a.k;
  if (!(t > 0.0)) { t = 1.0; s.k = 1; }  // no temperature: the first of the largest
  if (s.p <= 0.0) { s.p = 1.0; s.k = 1; }
  s.sc = fmin(1.4426950408889634074 / t, 1e300);
  s.least = mp > 0.0 ? fmin(mp, 1.0) * UNIT : 0.0;
  s.u = a.u[r];
  return s;
}
// the integer that the kept mass has to reach: mass > u * total
__device__ __forceinline__ u64 draw_at(float uf, u64 total) {
  const double u = uf > 0.0f ? fmin((double)uf, 1.0 - 1.0 / 9007199254740992.0) : 0.0;  // (NaN: 0)
  const u64 d = (u64)(u * (double)total);
  return d < total ? d + 1 : total;
}
// ceil(share of total): a member is kept whose mass before it is < share * total, so the prefix is the shortest whose mass reaches this
__device__ __forceinline__ u64 share_of(double share, u64 total) {
  const u64 need = (u64)ceil(share * (double)total);
  return need > total ? total : need < 1 ? 1 : need;
}
__device__ __forceinline__ float logp_of(uint32_t key, double m, double sc, bool inf_row, u64 total) {
  return (float)((inf_row ? 0.0 : ((double)score_of(key) - m) * (sc * 0.693147180559945309417)) - log((double)total / UNIT));
}

// halfway between two keys: by value for the first steps (scores spread evenly by value), then by bits, which ends for certain
__device__ __forceinline__ uint32_t middle(uint32_t lo, uint32_t hi, int step) {
  if (step < 16) {
    const uint32_t v = key_of(0.5f * score_of(lo) + 0.5f * score_of(hi - 1));
    if (v > lo && v < hi) return v;
  }
  return lo + (hi - lo) / 2;
}

// ---------------------------------------------------------------------------------------------------- rows of up to 64 E scores
// A lane holds E neighbours, so lanes are in index order.
template <class T, int E> __global__ __launch_bounds__(256) void k_sample_wave(Args a, int rows) {
  const int lane = threadIdx.x & 63, n = a.n;
  const int64_t r = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (r >= rows) return;
  const T *row = (const T *)a.scores + r * a.stride;
  const uint8_t *legal = a.legal ? a.legal + r * a.legal_stride : nullptr;
  const Setting st = setting_of(a, r);
  const int i0 = lane * E;
  uint32_t key[E], kmax = KEY_NONE, kmin = 0xFFFFFFFFu;
#pragma unroll
  for (int j = 0; j < E; ++j) key[j] = i0 + j < n ? key_of(to_f32(row[i0 + j])) : KEY_NONE;
  if (legal) {
#pragma unroll
    for (int j = 0; j < E; ++j)
      if (i0 + j < n && legal[i0 + j] == 0) key[j] = KEY_NONE;
  }
  int left = 0;
#pragma unroll
  for (int j = 0; j < E; ++j) {
    const bool on = key[j] != KEY_NONE;
    kmax = key[j] > kmax ? key[j] : kmax;
    kmin = on && key[j] < kmin ? key[j] : kmin;
    left += __popcll(__ballot(on));
  }
  if (left == 0) {
    if (lane == 0) {
      a.actions[r] = -1;
      if (a.logp) a.logp[r] = -INFINITY;
    }
    return;
  }
  kmax = wave_max(kmax);
  const bool inf_row = kmax == KEY_PINF;
  const double m = inf_row ? 0.0 : (double)score_of(kmax);
  // the first `take` (in index order) of the scores equal to `tie`, and what is above it, stay
  auto keep = [&](uint32_t tie, int take) {
    uint32_t eq = 0;
#pragma unroll
    for (int j = 0; j < E; ++j) eq += key[j] == tie;
    uint32_t before = wave_scan(eq) - eq;
#pragma unroll
    for (int j = 0; j < E; ++j) {
      const bool is = key[j] == tie;
      if (key[j] < tie || (is && before >= (uint32_t)take)) key[j] = KEY_NONE;
      before += is;
    }
  };
  const bool cut_k = st.k > 0 && st.k < left, cut_p = st.p < 1.0;
  if (cut_k || cut_p) kmin = ~wave_max(~kmin);
  if (cut_k) {  // count(>= lo) > k > count(>= hi), or the exact count
    uint32_t lo = kmin, hi = kmax + 1;
    int above = 0;
    bool exact = false;
    for (int step = 0; hi - lo > 1; ++step) {
      const uint32_t mid = middle(lo, hi, step);
      int c = 0;
#pragma unroll
      for (int j = 0; j < E; ++j) c += __popcll(__ballot(key[j] >= mid));
      if (c > st.k) lo = mid;
      else { hi = mid; above = c; }
      if (c == st.k) { exact = true; break; }
    }
    if (exact) keep(hi - 1, 0);
    else keep(lo, st.k - above);
    left = st.k;
  }
  u64 w[E];
  constexpr int SIDE = E < 4 ? E : 4;
#pragma unroll
  for (int j = 0; j < E; j += SIDE) weights<SIDE>(key + j, m, st.sc, inf_row, w + j);
  if (cut_p) {  // mass(>= lo) reaches the share, mass(>= hi) does not
    u64 s = 0;
#pragma unroll
    for (int j = 0; j < E; ++j) s += w[j];
    const u64 need = share_of(st.p, wave_sum(s));
    uint32_t lo = kmin, hi = kmax + 1;
    u64 above = 0;
    int c_lo = left, c_hi = 0;
    for (int step = 0; hi - lo > 1 && c_lo - c_hi > 1; ++step) {
      const uint32_t mid = middle(lo, hi, step);
      u64 s = 0;
      int c = 0;
#pragma unroll
      for (int j = 0; j < E; ++j) {
        const bool in = key[j] >= mid;
        s += in ? w[j] : 0;
        c += __popcll(__ballot(in));
      }
      s = wave_sum(s);
      if (s >= need) { lo = mid; c_lo = c; }
      else { hi = mid; above = s; c_hi = c; }
    }
    if (hi - lo > 1) keep(lo, 0x7FFFFFFF);  // one score in between: the last member
    else {
      const u64 each = weight(lo, m, st.sc, inf_row), take = (need - above + each - 1) / each;
      keep(lo, take < 0x7FFFFFFF ? (int)take : 0x7FFFFFFF);
    }
  }
  u64 mine = 0;
#pragma unroll
  for (int j = 0; j < E; ++j) {
    if (key[j] == KEY_NONE || (double)w[j] < st.least) w[j] = 0;
    mine += w[j];
  }
  const u64 incl = wave_scan(mine), total = lane_of(incl, 63), need = draw_at(st.u, total);
  if (incl >= need && incl - mine < need) {
    u64 run = incl - mine;
    int at = 0;
    uint32_t at_key = key[0];
#pragma unroll
    for (int j = 0; j < E; ++j) {
      if (run < need && run + w[j] >= need) { at = j; at_key = key[j]; }
      run += w[j];
    }
    a.actions[r] = i0 + at;
    if (a.logp) a.logp[r] = logp_of(at_key, m, st.sc, inf_row, total);
  }
}

// ---------------------------------------------------------------------------------------------------- longer rows
// The row as the workgroup sees it: vectors of 16 bytes, vector v of thread t holds the scores from (v * NT + t) * V on; a walk reads
// one vector ahead.  (Held in registers instead, every walk unrolls over all vectors: 20,000 instructions, and 1,024 threads spill.)
// Masked scores and those behind the row's end are NaN.
template <class T, int NT> struct Row {
  static constexpr int V = 16 / sizeof(T), N = Word<T>::N;
  const T *s;
  const uint8_t *legal;
  int n, tid, walks;

  __device__ __forceinline__ u32x4 read(int v) const {
    const int i = (v * NT + tid) * V;
    u32x4 w;
    if (i + V <= n) __builtin_memcpy(&w, s + i, 16);
    else {  // the row's last vector, and those behind it: every load at once, from inside the row
      T e[V];
#pragma unroll
      for (int j = 0; j < V; ++j) e[j] = s[min(i + j, n - 1)];
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (i + j >= n) from_f32(NAN, e[j]);
      __builtin_memcpy(&w, e, 16);
    }
    if (legal) {
      uint8_t on[V];
      if (i + V <= n) __builtin_memcpy(on, legal + i, V);
      else {
#pragma unroll
        for (int j = 0; j < V; ++j) on[j] = legal[min(i + j, n - 1)];
      }
#pragma unroll
      for (int j = 0; j < V; ++j) w[j / N] |= on[j] ? 0u : N == 1 ? 0xFFFFFFFFu : 0xFFFFu << (16 * (j % N));  // (all ones: a NaN of any type)
    }
    return w;
  }
  // f(keys of a vector, index of its first score, vector), all lanes together.  (Four vectors ahead instead of one gains nothing: a walk
  // is bound by its instructions.)
  template <class F> __device__ __forceinline__ void walk(F f) const {
    u32x4 next = read(0);
    for (int v = 0; v < walks; ++v) {
      const u32x4 w = next;
      if (v + 1 < walks) next = read(v + 1);
      uint32_t k[V];
#pragma unroll
      for (int j = 0; j < V; ++j) k[j] = key_of(Word<T>::get(w[j / N], j % N));
      f(k, (v * NT + tid) * V, v);
    }
  }
};

// a listed score: its place in the order as one number (key, then the lower index first), and its mass
struct alignas(16) Member {
  u64 rank, w;
  __device__ __forceinline__ uint32_t key() const { return (uint32_t)(rank >> 32); }
  __device__ __forceinline__ int idx() const { return (int)~(uint32_t)rank; }
};

template <int NT> struct Shared {
  u64 hist[BINS];
  u64 part[NT / 64];
  uint32_t kmax[NT / 64], kmin[NT / 64];
  u64 base, value;
  Member list[LIST];
  Member end;
  u64 end_upto;
  int32_t bin, count, end_idx;
  uint32_t reached;
};

struct Limit {  // the last member of a prefix of the order
  uint32_t key;
  int32_t idx;
  __device__ __forceinline__ bool has(uint32_t k, int i) const { return k > key || (k == key && i <= idx); }
};

// Where the running sum of hist (bins in order) first reaches `need`: sh.bin (BINS: nowhere), sh.base = the sum before that bin,
// sh.value = the bin's own.
template <int NT> __device__ __forceinline__ void find_bin(Shared<NT> &sh, u64 need, int tid) {
  constexpr int PER = BINS / NT;
  u64 mine = 0;
#pragma unroll
  for (int j = 0; j < PER; ++j) mine += sh.hist[tid * PER + j];
  const int lane = tid & 63, wave = tid >> 6;
  const u64 incl = wave_scan(mine);
  if (lane == 63) sh.part[wave] = incl;
  if (tid == 0) sh.bin = BINS;
  __syncthreads();
  u64 run = incl - mine;
  for (int w = 0; w < wave; ++w) run += sh.part[w];
  if (run < need && run + mine >= need) {
    for (int j = 0; j < PER; ++j) {
      const u64 v = sh.hist[tid * PER + j];
      if (run + v >= need) {
        sh.bin = tid * PER + j;
        sh.base = run;
        sh.value = v;
        break;
      }
      run += v;
    }
  }
  __syncthreads();
}

// Appends the keys of a vector that bits of `on` name: one addition to the count a wave.  Called by all lanes; beyond LIST the count goes
// on and nothing is stored.
template <int V, int NT> __device__ __forceinline__ void append(Shared<NT> &sh, uint32_t on, const uint32_t *key, int idx) {
  if (__ballot(on != 0) == 0) return;
  const uint32_t mine = __popc(on), incl = wave_scan(mine);
  int at = 0;
  if ((threadIdx.x & 63) == 63) at = atomicAdd(&sh.count, (int)incl);
  at = __builtin_amdgcn_readlane(at, 63) + (int)(incl - mine);
#pragma unroll
  for (int j = 0; j < V; ++j)
    if ((on >> j) & 1) {
      if (at < LIST) sh.list[at].rank = ((u64)key[j] << 32) | (uint32_t)~(idx + j);
      ++at;
    }
}

template <int NT> __device__ __forceinline__ u64 block_sum(Shared<NT> &sh, u64 v, int tid) {
  v = wave_sum(v);
  if ((tid & 63) == 0) sh.part[tid >> 6] = v;
  __syncthreads();
  v = 0;
  for (int w = 0; w < NT / 64; ++w) v += sh.part[w];
  __syncthreads();
  return v;
}

// Where the running sum of the list's masses, in the order that `ahead` tells and `bin_of` follows, first reaches need (at most their
// sum): sh.end, and the sum up to and with it in sh.end_upto.  A histogram, then the members of one bin, each of which sums what of
// them lies ahead of it.
template <int NT, class B, class A> __device__ __forceinline__ void list_find(Shared<NT> &sh, int c, u64 need, int tid, B bin_of, A ahead) {
  for (int i = tid; i < BINS; i += NT) sh.hist[i] = 0;
  if (tid == 0) sh.count = 0;
  __syncthreads();
  for (int e = tid; e < c; e += NT) {
    const Member m = sh.list[e];
    if (m.w) atomicAdd(&sh.hist[bin_of(m)], m.w);
  }
  __syncthreads();
  find_bin<NT>(sh, need, tid);
  const int b = sh.bin;
  const u64 base = sh.base;
  Member *own = (Member *)sh.hist;  // (the sums have been read)
  static_assert(sizeof(Member) * LIST <= sizeof(sh.hist), "a bin's members fit the histogram's memory");
  for (int e = tid; e < c; e += NT) {
    const Member m = sh.list[e];
    if (m.w && bin_of(m) == b) own[atomicAdd(&sh.count, 1)] = m;
  }
  __syncthreads();
  const int n = sh.count;
  for (int e = tid; e < n; e += NT) {
    const Member me = own[e];
    u64 upto = base + me.w;
#pragma unroll 4
    for (int x = 0; x < n; ++x) {
      const Member o = own[x];
      upto += ahead(o, me) ? o.w : 0;
    }
    if (upto >= need && upto - me.w < need) { sh.end = me; sh.end_upto = upto; }  // (one member)
  }
  __syncthreads();
}

// The shortest prefix of `in` (itself a prefix of the order) whose count reaches `need`, or (MASS) whose mass reaches the share
// `frac` of `in`'s mass.  A histogram linear in the score, then a list of the bin found; where that does not fit (thousands of nearly
// equal scores), histograms over their keys, 11 bits at a time, until a bin is one key, whose equal scores are cut by index.
template <bool MASS, int NT, class H>
__device__ __forceinline__ Limit cut(const H &row, Shared<NT> &sh, Limit in, uint32_t kmax, uint32_t kmin, double m, double sc, bool inf_row, u64 need, double frac) {
  constexpr int V = H::V;
  const int tid = row.tid, lane = tid & 63, wave = tid >> 6;
  const float top = score_of(kmax);
  float span = top - score_of(kmin);
  if (MASS) span = fminf(span, (float)(45.0 / sc));  // below 2^-45 of the largest there is no mass
  const float scale = (float)BINS / span;
  uint32_t khi = kmax, klo = KEY_NONE + 1;
  u64 base = 0;
  bool linear = span > 0.0f && span < INFINITY && scale < INFINITY && kmax - kmin >= (uint32_t)BINS;
  if (!linear) klo = kmin;
  auto bin_of = [&](uint32_t k) { return (int)fminf((top - score_of(k)) * scale, (float)(BINS - 1)); };
  for (;;) {
    for (int i = tid; i < BINS; i += NT) sh.hist[i] = 0;
    if (tid == 0) sh.count = 0;
    __syncthreads();
    const int bits = 32 - __clz((int)(khi - klo) | 1), shift = bits > 11 ? bits - 11 : 0;
    row.walk([&](const uint32_t *k, int i, int) {
      bool on[V];
      u64 w[V];
#pragma unroll
      for (int j = 0; j < V; ++j) on[j] = k[j] != KEY_NONE && k[j] <= khi && k[j] >= klo && in.has(k[j], i + j);
      if (MASS) weights<V>(k, m, sc, inf_row, w);
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (on[j] && (!MASS || w[j])) atomicAdd(&sh.hist[linear ? bin_of(k[j]) : (int)((khi - k[j]) >> shift)], MASS ? w[j] : 1);
    });
    __syncthreads();
    if (MASS && frac > 0.0) {  // the first histogram holds the whole mass of `in`: the target is a share of it
      u64 s = 0;
      for (int i = tid; i < BINS; i += NT) s += sh.hist[i];
      s = block_sum<NT>(sh, s, tid);
      need = share_of(frac, s);
      frac = 0.0;
    }
    find_bin<NT>(sh, need - base, tid);
    if (sh.bin >= BINS) return in;  // never reached: nothing is cut
    const int b = sh.bin;
    const u64 value = sh.value;
    base += sh.base;
    __syncthreads();
    if (linear) {
      // the scores of that bin: their list, and the range of their keys
      uint32_t hi = KEY_NONE, lo = 0xFFFFFFFFu;
      row.walk([&](const uint32_t *k, int i, int) {
        uint32_t on = 0;
#pragma unroll
        for (int j = 0; j < V; ++j)
          if (k[j] != KEY_NONE && in.has(k[j], i + j) && bin_of(k[j]) == b) {
            hi = k[j] > hi ? k[j] : hi;
            lo = k[j] < lo ? k[j] : lo;
            on |= 1u << j;
          }
        append<V, NT>(sh, on, k, i);
      });
      hi = wave_max(hi);
      lo = ~wave_max(~lo);
      if (lane == 0) { sh.kmax[wave] = hi; sh.kmin[wave] = lo; }
      __syncthreads();
      const int c = sh.count;
      if (c <= LIST) {
        for (int e = tid; e < c; e += NT) sh.list[e].w = MASS ? weight(sh.list[e].key(), m, sc, inf_row) : 1;
        __syncthreads();
        uint32_t first_key = KEY_NONE;
        for (int w = 0; w < NT / 64; ++w) first_key = max(first_key, sh.kmax[w]);
        const float first = score_of(first_key), fine = fminf((float)BINS * scale, 3e38f);
        list_find<NT>(sh, c, need - base, tid, [&](const Member &x) { return (int)fminf((first - score_of(x.key())) * fine, (float)(BINS - 1)); },
                      [](const Member &x, const Member &me) { return x.rank > me.rank; });
        return Limit{sh.end.key(), sh.end.idx()};
      }
      khi = KEY_NONE;
      klo = 0xFFFFFFFFu;
      for (int w = 0; w < NT / 64; ++w) { khi = sh.kmax[w] > khi ? sh.kmax[w] : khi; klo = sh.kmin[w] < klo ? sh.kmin[w] : klo; }
      __syncthreads();
      linear = false;
      continue;
    }
    if (shift > 0) {
      const uint32_t top_key = khi - ((uint32_t)b << shift), width = (1u << shift) - 1u;
      klo = top_key - klo > width ? top_key - width : klo;
      khi = top_key;
      continue;
    }
    // one key: how many of its equal scores come in
    const uint32_t tk = khi - (uint32_t)b;
    const u64 each = MASS ? weight(tk, m, sc, inf_row) : 1, ties = value / each;  // (a bin that is reached holds mass)
    const u64 take = (need - base + each - 1) / each;
    if (take >= ties) return Limit{tk, tk == in.key ? in.idx : 0x7FFFFFFF};
    // the index of the take-th equal score: counted in index order, a vector of every thread at a time
    u64 seen = 0;
    row.walk([&](const uint32_t *k, int i, int) {
      if (seen >= take) return;  // (uniform)
      uint32_t mine = 0;
#pragma unroll
      for (int j = 0; j < V; ++j) mine += k[j] == tk;
      const uint32_t incl = wave_scan(mine);
      if (lane == 63) sh.part[wave] = incl;
      __syncthreads();
      u64 before = seen + incl - mine, all = 0;
      for (int w = 0; w < NT / 64; ++w) { before += w < wave ? sh.part[w] : 0; all += sh.part[w]; }
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (k[j] == tk && ++before == take) sh.end_idx = i + j;
      seen += all;
      __syncthreads();
    });
    return Limit{tk, sh.end_idx};
  }
}

template <class T, int NT> __global__ __launch_bounds__(NT) void k_sample_block(Args a) {
  __shared__ Shared<NT> sh;
  constexpr int WAVES = NT / 64, V = 16 / sizeof(T);
  const int64_t r = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = a.n, walks = (n + NT * V - 1) / (NT * V);
  const Row<T, NT> row{(const T *)a.scores + r * a.stride, a.legal ? a.legal + r * a.legal_stride : nullptr, n, tid, walks};
  const Setting st = setting_of(a, r);
  // the largest of every thread's vectors v, v + G, ..: 1,024 numbers, whatever the workgroup
  constexpr int G = 1024 / NT;
  uint32_t kmax = KEY_NONE, own_max[G];
#pragma unroll
  for (int q = 0; q < G; ++q) own_max[q] = KEY_NONE;
  row.walk([&](const uint32_t *k, int, int v) {
    uint32_t most = k[0];
#pragma unroll
    for (int j = 1; j < V; ++j) most = k[j] > most ? k[j] : most;
#pragma unroll
    for (int q = 0; q < G; ++q)
      if ((v & (G - 1)) == q) own_max[q] = max(own_max[q], most);
  });
#pragma unroll
  for (int q = 0; q < G; ++q) kmax = max(kmax, own_max[q]);
  kmax = wave_max(kmax);
  if (lane == 0) sh.kmax[wave] = kmax;
  __syncthreads();
  for (int w = 0; w < WAVES; ++w) kmax = sh.kmax[w] > kmax ? sh.kmax[w] : kmax;
  __syncthreads();
  if (kmax == KEY_NONE) {  // nothing legal
    if (tid == 0) {
      a.actions[r] = -1;
      if (a.logp) a.logp[r] = -INFINITY;
    }
    return;
  }
  const bool inf_row = kmax == KEY_PINF;
  const double m = inf_row ? 0.0 : (double)score_of(kmax);
  const bool cut_k = st.k > 0 && st.k < n, cut_p = st.p < 1.0;
  if ((cut_k || cut_p) && !(cut_k && st.k > LIST)) {
    // the largest key that nine sixteenths of those numbers reach, or, for the top k, that k of them do (all legal scores, if too few hold any)
    uint32_t *tops = (uint32_t *)sh.hist;
#pragma unroll
    for (int q = 0; q < G; ++q) tops[q * NT + tid] = own_max[q];
    if (tid == 0) sh.count = 0;
    __syncthreads();
    if (wave == 0) {
      uint32_t top[16], lo = 0xFFFFFFFFu, hi = kmax + 1;
      const int share = min(walks, G) * (NT * 9 / 16), want = cut_k && st.k < share ? st.k : share;
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        top[j] = tops[j * 64 + lane];
        lo = min(lo, top[j]);
      }
      lo = ~wave_max(~lo);
      for (int step = 0; hi - lo > 1; ++step) {
        const uint32_t mid = lo == KEY_NONE ? lo + (hi - lo) / 2 : middle(lo, hi, step);
        int c = 0;
#pragma unroll
        for (int j = 0; j < 16; ++j) c += __popcll(__ballot(top[j] >= mid));
        if (c >= want) lo = mid;
        else hi = mid;
        if (c == want) break;
      }
      if (lane == 0) sh.reached = lo == KEY_NONE ? KEY_NONE + 1 : lo;
    }
    __syncthreads();
    const uint32_t reached = sh.reached;
    // The mass of the row to within a share OFF, from f32 exponentials: (s - m) sc carries three roundings of 2^-24 of itself, at most 40
    // before a weight is below 2^-40 (and all such together below 2^-21), the exponential 2^-22.  Where that does not settle where the
    // prefix ends (a few rows in a hundred), the mass is summed exactly.
    constexpr double OFF = 0x1p-17;
    const float mf = score_of(kmax), scf = (float)st.sc;
    // (a factor below 2^-120, of a temperature next to infinity, would meet infinite differences)
    const bool rough = !cut_k && !inf_row && scf < 1e30f && scf > 0x1p-120f;
    double part = 0.0;
    row.walk([&](const uint32_t *k, int i, int) {
      uint32_t on = 0;
#pragma unroll
      for (int j = 0; j < V; ++j) on |= k[j] >= reached ? 1u << j : 0;
      append<V, NT>(sh, on, k, i);
      if (rough) {
        float w = 0.0f;
#pragma unroll
        for (int j = 0; j < V; ++j) w += __builtin_amdgcn_exp2f((score_of(k[j]) - mf) * scf);
        part += (double)w;
      }
    });
    u64 mass = block_sum<NT>(sh, (u64)(part * UNIT), tid);
    int c = sh.count;
    __syncthreads();
    bool ends = c <= LIST && (!cut_k || c >= st.k || reached == KEY_NONE + 1);  // the prefix ends within the list
    if (ends) {
      const float top = score_of(kmax), scale = fminf((float)BINS / (top - score_of(reached)), 3e38f);  // (NaN and infinity: the first or the last bin)
      auto in_order = [](const Member &x, const Member &me) { return x.rank > me.rank; };
      auto by_score = [&](const Member &x) { return (int)fminf((top - score_of(x.key())) * scale, (float)(BINS - 1)); };
      u64 last = 0;  // the place of the prefix's last member
      if (cut_k && c > st.k) {
        for (int e = tid; e < c; e += NT) sh.list[e].w = 1;
        __syncthreads();
        list_find<NT>(sh, c, (u64)st.k, tid, by_score, in_order);
        last = sh.end.rank;
      }
      u64 sum = 0;
      for (int e = tid; e < c; e += NT) sum += sh.list[e].w = sh.list[e].rank >= last ? weight(sh.list[e].key(), m, st.sc, inf_row) : 0;
      sum = block_sum<NT>(sh, sum, tid);
      if (cut_p) {
        u64 need = share_of(st.p, sum);
        bool found = false;
        if (!cut_k && rough) {
          need = share_of(st.p, (u64)((double)mass * (1.0 - OFF)));
          ends = sum >= need;
          if (ends) {
            list_find<NT>(sh, c, need, tid, by_score, in_order);
            found = share_of(st.p, (u64)((double)mass * (1.0 + OFF))) <= sh.end_upto;
          }
        }
        if (ends && !found) {
          if (!cut_k) {
            mass = 0;
            row.walk([&](const uint32_t *k, int, int) {
              u64 w[V];
              weights<V>(k, m, st.sc, inf_row, w);
#pragma unroll
              for (int j = 0; j < V; ++j) mass += w[j];
            });
            need = share_of(st.p, block_sum<NT>(sh, mass, tid));
            ends = sum >= need;
          }
          if (ends) list_find<NT>(sh, c, need, tid, by_score, in_order);
        }
        last = sh.end.rank;
      }
      if (ends) {
        sum = 0;
        for (int e = tid; e < c; e += NT) {
          Member &x = sh.list[e];
          if (x.rank < last || (double)x.w < st.least) x.w = 0;
          sum += x.w;
        }
        const u64 total = block_sum<NT>(sh, sum, tid);
        const int shift = 32 - __clz((n - 1) | 1) > 11 ? 32 - __clz((n - 1) | 1) - 11 : 0;
        list_find<NT>(sh, c, draw_at(st.u, total), tid, [&](const Member &x) { return x.idx() >> shift; },
                      [](const Member &x, const Member &me) { return x.idx() < me.idx(); });
        if (tid == 0) {
          a.actions[r] = sh.end.idx();
          if (a.logp) a.logp[r] = logp_of(sh.end.key(), m, st.sc, inf_row, total);
        }
        return;
      }
    }
    __syncthreads();
  }
  Limit lim{KEY_NONE, -1};
  uint32_t kmin = 0xFFFFFFFFu;
  if (cut_k || cut_p) {
    row.walk([&](const uint32_t *k, int, int) {
#pragma unroll
      for (int j = 0; j < V; ++j) kmin = min(kmin, k[j] - (KEY_NONE + 1));  // (KEY_NONE wraps to the top)
    });
    kmin = ~wave_max(~kmin);
    if (lane == 0) sh.kmin[wave] = kmin;
    __syncthreads();
    for (int w = 0; w < WAVES; ++w) kmin = min(kmin, sh.kmin[w]);
    kmin += KEY_NONE + 1;
    __syncthreads();
  }
  if (cut_k) {
    lim = cut<false, NT>(row, sh, lim, kmax, kmin, m, st.sc, inf_row, (u64)st.k, 0.0);
    __syncthreads();
  }
  if (cut_p) {
    lim = cut<true, NT>(row, sh, lim, kmax, kmin, m, st.sc, inf_row, 0, st.p);
    __syncthreads();
  }
  // kept mass of every wave's share of every vector, in index order: walks * WAVES sums, at most 2^19 / (64 V) = 2,048
  auto kept_of = [&](const uint32_t *k, int i, u64 *w) {  // -> their sum
    weights<V>(k, m, st.sc, inf_row, w);
    u64 s = 0;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      if (!lim.has(k[j], i + j) || (double)w[j] < st.least) w[j] = 0;
      s += w[j];
    }
    return s;
  };
  row.walk([&](const uint32_t *k, int i, int v) {
    u64 w[V];
    const u64 s = wave_sum(kept_of(k, i, w));
    if (lane == 0) sh.hist[v * WAVES + wave] = s;
  });
  const int sums = walks * WAVES;
  for (int i = sums + tid; i < BINS; i += NT) sh.hist[i] = 0;
  __syncthreads();
  u64 total = 0;
  for (int i = lane; i < sums; i += 64) total += sh.hist[i];
  total = wave_sum(total);
  const u64 need = draw_at(st.u, total);
  find_bin<NT>(sh, need, tid);  // (a bin is found: need <= total)
  if (sh.bin % WAVES != wave) return;
  const int v = sh.bin / WAVES;
  const u32x4 words = row.read(v);
  uint32_t keys[V];
  u64 w[V];
#pragma unroll
  for (int j = 0; j < V; ++j) keys[j] = key_of(Word<T>::get(words[j / Word<T>::N], j % Word<T>::N));
  const u64 mine = kept_of(keys, (v * NT + tid) * V, w);
  u64 run = sh.base + wave_scan(mine) - mine;
  if (run < need && run + mine >= need) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      if (run < need && run + w[j] >= need) {
        a.actions[r] = (v * NT + tid) * V + j;
        if (a.logp) a.logp[r] = logp_of(keys[j], m, st.sc, inf_row, total);
      }
      run += w[j];
    }
  }
}

// The kernel that holds a row of n scores.  Measured (us; bf16, top p 0.9 alone / with top k 40):
//   a wave for up to 1,024: 8,192 x 1,024 f32 52 / 58, a workgroup of 256 86 / 92; 32 scores a lane at 8,192 x 2,048 115 / 124, the workgroup 104 / 100
//   1,024 threads or 256, four of which share a CU where two of those do: 64 x 5,000 42 / 23 or 28 / 22, 1 x 20,000 62 / 24 or 75 / 20,
//   1 x 65,537 119 / 26 or 194 / 42, 512 x 20,000 138 / 47 or 94 / 30, 512 x 65,537 264 / 62 or 254 / 49, 2,048 x 65,537 1,044 / 240 or 774 / 144,
//   512 x 131,072 422 / 77 or 452 / 71 (245 or 363 at temperature 0.7): 256 where rows are short, or fill the card and are not the longest
template <class T> static void launch_rows(const Args &a, int rows, hipStream_t s) {
  const dim3 four((rows + 3) / 4), one(rows);
  if (a.n <= 64) hipLaunchKernelGGL((k_sample_wave<T, 1>), four, dim3(256), 0, s, a, rows);
  else if (a.n <= 128) hipLaunchKernelGGL((k_sample_wave<T, 2>), four, dim3(256), 0, s, a, rows);
  else if (a.n <= 256) hipLaunchKernelGGL((k_sample_wave<T, 4>), four, dim3(256), 0, s, a, rows);
  else if (a.n <= 512) hipLaunchKernelGGL((k_sample_wave<T, 8>), four, dim3(256), 0, s, a, rows);
  else if (a.n <= 1024) hipLaunchKernelGGL((k_sample_wave<T, 16>), four, dim3(256), 0, s, a, rows);
  else if (a.n <= 8192 || (rows >= 512 && a.n <= 98304)) hipLaunchKernelGGL((k_sample_block<T, 256>), one, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((k_sample_block<T, 1024>), one, dim3(1024), 0, s, a);
}

// a launch holds fewer than 2^32 threads: 2^21 rows at a time
template <class T> static void launch(Args a, int rows, hipStream_t s) {
  for (constexpr int MOST = 1 << 21;;) {
    const int m = rows < MOST ? rows : MOST;
    launch_rows<T>(a, m, s);
    if ((rows -= m) == 0) return;
    a.scores = (const T *)a.scores + m * a.stride;
    if (a.legal) a.legal += m * a.legal_stride;
    a.u += m;
    a.actions += m;
    if (a.logp) a.logp += m;
    if (a.t_rows) a.t_rows += m;
    if (a.p_rows) a.p_rows += m;
    if (a.mp_rows) a.mp_rows += m;
    if (a.k_rows) a.k_rows += m;
  }
}

}  // namespace azsample

extern "C" int az_sample_actions(int32_t dtype, int32_t rows, int32_t n, const void *scores_dev, int64_t row_stride, const uint8_t *legal_dev,
                                 int64_t legal_stride, const float *uniforms_dev, const float *temperature_dev, double temperature,
                                 const int32_t *top_k_dev, int32_t top_k, const float *top_p_dev, double top_p, const float *min_p_dev,
                                 double min_p, int32_t *actions_dev, float *logprobs_dev, void *stream) {
  using namespace azsample;
  if (dtype != AZ_NN_F32 && dtype != AZ_NN_BF16 && dtype != AZ_NN_F16) return fail(AZ_EINVAL, "sample: unknown dtype");
  if (rows < 0 || n < 1 || n > MAX_N) return fail(AZ_EINVAL, "sample: rows >= 0 and 1 <= n <= 524,288");
  if (rows == 0) return AZ_OK;
  if (!scores_dev || !uniforms_dev || !actions_dev) return fail(AZ_EINVAL, "sample: null argument");
  if (row_stride < 0 || (legal_dev && legal_stride < 0)) return fail(AZ_EINVAL, "sample: negative row stride");  // (0: one row for all draws)
  if (misaligned(scores_dev, dtype == AZ_NN_F32 ? 4 : 2) || misaligned(uniforms_dev, 4) || misaligned(temperature_dev, 4) ||
      misaligned(top_k_dev, 4) || misaligned(top_p_dev, 4) || misaligned(min_p_dev, 4) || misaligned(actions_dev, 4) || misaligned(logprobs_dev, 4))
    return fail(AZ_EINVAL, "sample: misaligned pointer");
  if (!temperature_dev && !(temperature >= 0.0)) return fail(AZ_EINVAL, "sample: temperature >= 0");
  if (!top_p_dev && !(top_p >= 0.0)) return fail(AZ_EINVAL, "sample: top_p >= 0");
  if (!min_p_dev && !(min_p >= 0.0 && min_p <= 1.0)) return fail(AZ_EINVAL, "sample: 0 <= min_p <= 1");
  hipStream_t s = (hipStream_t)stream;
  DeviceGuard guard(s);
  if (!guard.ok) return fail(AZ_EHIP, "sample: cannot select the stream's device");
  Args a{scores_dev, legal_dev, uniforms_dev, temperature_dev, top_p_dev, min_p_dev, top_k_dev, actions_dev, logprobs_dev,
         row_stride, legal_stride, temperature, top_p, min_p, top_k, n};
  if (dtype == AZ_NN_F32) launch<float>(a, rows, s);
  else if (dtype == AZ_NN_BF16) launch<bf16_t>(a, rows, s);
  else launch<f16_t>(a, rows, s);
  return launched("k_sample");
}
