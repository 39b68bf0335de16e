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
// The kept set is a prefix of the order, so it is described by its last member (key, index), and no row is ever sorted: the
// prefix's end is found from histograms over the 32-bit order-preserving image of the score.
#include "az_ops.hip.h"

namespace azsample {

using namespace azops;
typedef unsigned long long u64;

constexpr int MAX_N = 1 << 19, BINS = 2048, NT = 256, WAVES = NT / 64;
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

// 2^44 exp((s - m) / T) rounded to an integer; sc = log2(e) / T.  2^f on [-1/2, 1/2] by its Taylor polynomial of degree 12
// (remainder below 2^-51); scores of +inf share the whole mass.
__device__ __forceinline__ u64 weight(uint32_t key, double m, double sc, bool inf_row) {
  if (key == KEY_NONE) return 0;
  if (inf_row) return key == KEY_PINF ? (u64)UNIT : 0;
  double y = ((double)score_of(key) - m) * sc;
  y = y < -100.0 ? -100.0 : y;
  const double kf = rint(y), f = (y - kf) * 0.693147180559945309417;
  double r = 1.0 / 479001600.0;
  r = fma(r, f, 1.0 / 39916800.0);
  r = fma(r, f, 1.0 / 3628800.0);
  r = fma(r, f, 1.0 / 362880.0);
  r = fma(r, f, 1.0 / 40320.0);
  r = fma(r, f, 1.0 / 5040.0);
  r = fma(r, f, 1.0 / 720.0);
  r = fma(r, f, 1.0 / 120.0);
  r = fma(r, f, 1.0 / 24.0);
  r = fma(r, f, 1.0 / 6.0);
  r = fma(r, f, 0.5);
  r = fma(r, f, 1.0);
  r = fma(r, f, 1.0);
  // 2^52 + w: the integer stands in the low mantissa bits, rounded to nearest even (w <= 2^44)
  return (u64)__double_as_longlong(ldexp(r, (int)kf + 44) + 4503599627370496.0) & 0xFFFFFFFFFFFFFull;
}

__device__ __forceinline__ u64 wave_sum(u64 v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) { const uint32_t x = __shfl_xor(v, o); v = x > v ? x : v; }
  return v;
}
__device__ __forceinline__ u64 wave_scan(u64 v, int lane) {  // inclusive
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) { const u64 x = __shfl_up(v, o); v += lane >= o ? x : 0; }
  return v;
}

struct Shared {
  u64 hist[BINS];
  u64 part[WAVES];
  uint32_t kmax[WAVES], kmin[WAVES];
  u64 base, value;
  int32_t bin, tie;
};

template <class T> struct Row {
  const T *s;
  const uint8_t *legal;
  __device__ __forceinline__ uint32_t key(int i) const { return legal != nullptr && legal[i] == 0 ? KEY_NONE : key_of(to_f32(s[i])); }
};

struct Limit {  // the last member of a prefix of the order
  uint32_t key;
  int32_t idx;
  __device__ __forceinline__ bool has(uint32_t k, int i) const { return k > key || (k == key && i <= idx); }
};

// Where the running sum of hist (bins in order) first reaches `need`: sh.bin (BINS: nowhere), sh.base = the sum before that bin,
// sh.value = the bin's own.
__device__ void find_bin(Shared &sh, u64 need, int tid) {
  constexpr int PER = BINS / NT;
  u64 mine = 0;
#pragma unroll
  for (int j = 0; j < PER; ++j) mine += sh.hist[tid * PER + j];
  const int lane = tid & 63, wave = tid >> 6;
  const u64 incl = wave_scan(mine, lane);
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

// The shortest prefix of `in` (itself a prefix of the order) whose count reaches `need`, or (MASS) whose mass reaches the share
// `frac` of `in`'s mass.  A prefix of the order keeps a member whose mass before it is < P: as masses are integers, that is the
// shortest prefix whose mass is >= ceil(P).  First a histogram linear in the score (spreads the atomics), then histograms over the keys of the bin found,
// 11 bits at a time, until a bin is one key; its equal scores are cut by index.
template <class T, bool MASS>
__device__ Limit cut(const Row<T> &row, int n, Shared &sh, Limit in, uint32_t kmax, uint32_t kmin, double m, double sc, bool inf_row,
                     u64 need, double frac, int tid) {
  const int lane = tid & 63, wave = tid >> 6;
  const float top = score_of(kmax);
  float span = top - score_of(kmin);
  if (MASS) span = fminf(span, (float)(45.0 / sc));  // below 2^-45 of the largest there is no mass
  const float scale = (float)BINS / span;
  uint32_t khi = kmax, klo = KEY_NONE + 1;
  u64 base = 0;
  bool linear = span > 0.0f && span < INFINITY && scale < INFINITY && kmax - kmin >= (uint32_t)BINS;
  if (!linear) klo = kmin;
  for (;;) {
    for (int i = tid; i < BINS; i += NT) sh.hist[i] = 0;
    __syncthreads();
    const int bits = 32 - __clz((int)(khi - klo) | 1), shift = bits > 11 ? bits - 11 : 0;
    for (int i = tid; i < n; i += NT) {
      const uint32_t k = row.key(i);
      if (k == KEY_NONE || k > khi || k < klo || !in.has(k, i)) continue;
      const int b = linear ? (int)fminf((top - score_of(k)) * scale, (float)(BINS - 1)) : (int)((khi - k) >> shift);
      const u64 v = MASS ? weight(k, m, sc, inf_row) : 1;
      if (v) atomicAdd(&sh.hist[b], v);
    }
    __syncthreads();
    if (MASS && frac > 0.0) {  // the first histogram holds the whole mass of `in`: the target is a share of it
      u64 s = 0;
      for (int i = tid; i < BINS; i += NT) s += sh.hist[i];
      s = wave_sum(s);
      if (lane == 0) sh.part[wave] = s;
      __syncthreads();
      s = 0;
      for (int w = 0; w < WAVES; ++w) s += sh.part[w];
      __syncthreads();
      need = (u64)ceil(frac * (double)s);  // frac < 1: at most the mass itself, but for the rounding
      need = need > s ? s : need < 1 ? 1 : need;
      frac = 0.0;
    }
    find_bin(sh, need - base, tid);
    if (sh.bin >= BINS) return in;  // never reached: nothing is cut
    const int b = sh.bin;
    const u64 before = base + sh.base, value = sh.value;
    __syncthreads();
    base = before;
    if (linear) {  // the keys of that bin
      uint32_t hi = KEY_NONE, lo = 0xFFFFFFFFu;
      for (int i = tid; i < n; i += NT) {
        const uint32_t k = row.key(i);
        if (k == KEY_NONE || k > khi || !in.has(k, i)) continue;
        if ((int)fminf((top - score_of(k)) * scale, (float)(BINS - 1)) != b) continue;
        hi = k > hi ? k : hi;
        lo = k < lo ? k : lo;
      }
      hi = wave_max(hi);
      lo = ~wave_max(~lo);
      if (lane == 0) { sh.kmax[wave] = hi; sh.kmin[wave] = lo; }
      __syncthreads();
      khi = KEY_NONE;
      klo = 0xFFFFFFFFu;
      for (int w = 0; w < WAVES; ++w) { khi = sh.kmax[w] > khi ? sh.kmax[w] : khi; klo = sh.kmin[w] < klo ? sh.kmin[w] : klo; }
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
    // the index of the take-th equal score: counted in index order
    if (tid == 0) sh.tie = -1;
    __syncthreads();
    u64 seen = 0;
    for (int i0 = 0; i0 < n; i0 += NT) {
      const int i = i0 + tid;
      const bool eq = i < n && row.key(i) == tk;
      const u64 mask = __ballot(eq);
      if (lane == 0) sh.part[wave] = (u64)__popcll(mask);
      __syncthreads();
      u64 mine = seen, all = 0;
      for (int w = 0; w < WAVES; ++w) { mine += w < wave ? sh.part[w] : 0; all += sh.part[w]; }
      mine += (u64)__popcll(mask & ((2ull << lane) - 1));
      if (eq && mine == take) sh.tie = i;
      seen += all;
      __syncthreads();
      if (seen >= take) break;
    }
    return Limit{tk, sh.tie};
  }
}

template <class T>
__global__ __launch_bounds__(NT) void k_sample_block(Args a) {
  __shared__ Shared sh;
  const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = a.n;
  const Row<T> row{(const T *)a.scores + (int64_t)r * a.stride, a.legal ? a.legal + (int64_t)r * a.legal_stride : nullptr};
  double t = a.t_rows ? (double)a.t_rows[r] : a.t, p = a.p_rows ? (double)a.p_rows[r] : a.p, mp = a.mp_rows ? (double)a.mp_rows[r] : a.mp;
  int k = a.k_rows ? a.k_rows[r] : a.k;
  if (!(t > 0.0)) { t = 1.0; k = 1; }  // no temperature: the first of the largest
  const double sc = fmin(1.4426950408889634074 / t, 1e300);
  uint32_t kmax = KEY_NONE, kmin = 0xFFFFFFFFu;
  for (int i = tid; i < n; i += NT) {
    const uint32_t key = row.key(i);
    if (key == KEY_NONE) continue;
    kmax = key > kmax ? key : kmax;
    kmin = key < kmin ? key : kmin;
  }
  kmax = wave_max(kmax);
  kmin = ~wave_max(~kmin);
  if (lane == 0) { sh.kmax[wave] = kmax; sh.kmin[wave] = kmin; }
  __syncthreads();
  for (int w = 0; w < WAVES; ++w) { kmax = sh.kmax[w] > kmax ? sh.kmax[w] : kmax; kmin = sh.kmin[w] < kmin ? sh.kmin[w] : kmin; }
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
  Limit lim{KEY_NONE, -1};
  if (k > 0 && k < n) lim = cut<T, false>(row, n, sh, lim, kmax, kmin, m, sc, inf_row, (u64)k, 0.0, tid);
  __syncthreads();
  if (p < 1.0) {
    if (p <= 0.0) lim = cut<T, false>(row, n, sh, lim, kmax, kmin, m, sc, inf_row, 1, 0.0, tid);
    else lim = cut<T, true>(row, n, sh, lim, kmax, kmin, m, sc, inf_row, 0, p, tid);
    __syncthreads();
  }
  const double least = mp > 0.0 ? fmin(mp, 1.0) * UNIT : 0.0;
  // kept mass of every tile of NT indices, in index order
  const int tiles = (n + NT - 1) / NT;
  auto kept = [&](int i) -> u64 {
    if (i >= n) return 0;
    const uint32_t key = row.key(i);
    if (key == KEY_NONE || !lim.has(key, i)) return 0;
    const u64 w = weight(key, m, sc, inf_row);
    return (double)w >= least ? w : 0;
  };
  for (int i = tid; i < BINS; i += NT) sh.hist[i] = 0;
  __syncthreads();
  for (int tile = 0; tile < tiles; ++tile) {
    const u64 s = wave_sum(kept(tile * NT + tid));
    if (lane == 0 && s) atomicAdd(&sh.hist[tile], s);
  }
  __syncthreads();
  u64 total = 0;
  for (int i = 0; i < tiles; i += 64) total += wave_sum(i + lane < tiles ? sh.hist[i + lane] : 0);
  const float uf = a.u[r];
  const double u = uf > 0.0f ? fmin((double)uf, 1.0 - 1.0 / 9007199254740992.0) : 0.0;  // (NaN: 0)
  const u64 drawn = (u64)(u * (double)total), need = drawn < total ? drawn + 1 : total;  // mass > u * total, in integers
  int tile = 0;
  u64 before = 0;
  while (before + sh.hist[tile] < need) before += sh.hist[tile++];  // (uniform; ends: need <= total)
  const int i = tile * NT + tid;
  const u64 w = kept(i);
  u64 incl = wave_scan(w, lane);
  if (lane == 63) sh.part[wave] = incl;
  __syncthreads();
  incl += before;
  for (int x = 0; x < wave; ++x) incl += sh.part[x];
  if (incl >= need && incl - w < need) sh.tie = i;
  __syncthreads();
  if (tid == 0) {
    const int at = sh.tie;
    a.actions[r] = at;
    if (a.logp) a.logp[r] = (float)((inf_row ? 0.0 : ((double)score_of(row.key(at)) - m) * (sc * 0.693147180559945309417)) - log((double)total / UNIT));
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
  if (dtype == AZ_NN_F32) hipLaunchKernelGGL(k_sample_block<float>, dim3(rows), dim3(NT), 0, s, a);
  else if (dtype == AZ_NN_BF16) hipLaunchKernelGGL(k_sample_block<bf16_t>, dim3(rows), dim3(NT), 0, s, a);
  else hipLaunchKernelGGL(k_sample_block<f16_t>, dim3(rows), dim3(NT), 0, s, a);
  return launched("k_sample");
}
