// az_norm.hip -- group norm with an activation over channels-last samples, forward and backward (gfx950).
//
//   a sample is (HW pixels, C channels), channels consecutive; group g = C / G consecutive channels of every pixel
//   xhat = (x - mean) rstd,  rstd = 1 / sqrt(var + eps),  z = xhat w + b (+ r),  y = act(z),  act: none, relu, silu
//   dz = dy act'(z);  dr = dz;  dw = sum dz xhat;  db = sum dz;
//   dx = rstd (dz w - mean_g(dz w) - xhat mean_g(dz w xhat))
//
// Bound by bytes: forward reads x (and r) and writes y, backward reads x, dy (and r) and writes dx (and dr).  A large copy reaches 5.04 TB/s
// on this card (reads and writes counted).  A sample whose channels fit a workgroup's registers is read once (k_gn_fwd_one, k_gn_bwd_one);
// a larger one is shared out over workgroups and read twice.  Measured:
//   1,024 x 128 x 15 x 15 f32, relu, residual: forward 77.5 us (354 MB: 4.6 TB/s), backward 117.5 us (590 MB: 5.0 TB/s) + 5.5 us for dw, db
//   16,384 x 64 x 15 x 15 bf16, relu, forward: 164 us (944 MB: 5.8 TB/s)
//   4 x 512 x 128 x 127 f16, silu, in chunks:  forward 13.9 + 4.4 + 22.9 us, backward 26.8 + 5.0 + 33.2 + 4.0 us (66.6 MB a tensor: the four
//                                              passes move 4.8, 5.8, 5.0 and 6.0 TB/s)
//   64 x 64 x 9 x 9 f32, relu:                 4.3 us, 4.8 + 3.1 us; the call is bound by the host (113 .. 120 us with autograd's own 72)
//   Slower than they could be (a group's vectors no power of two: in chunks; one or two channels: single elements, and one thread a group adds up):
//   1,024 x 192 x 15 x 15 f32 in 8 groups, relu: 314 us forward and backward; 16,384 x 1 x 15 x 15 bf16 forward 277 us (a floor of 3)
// Mean and variance come from f64 sums of x - p and (x - p)^2 in one pass, p the group's first value (of the sample's first pixel).  p is one
// of the m values, so (mean - p)^2 <= m var: the sums lose at most a factor of m of f64's 53 bits wherever the values lie (sums of x and x^2
// lose (mean / deviation)^2 of them), and a flat group has no variance at all.  The mean is kept as a pair of f32 for the subtraction,
// everything per element is f32, and each output is rounded once.  A relu's gradient hangs on the sign of z: where f32 cannot tell it, z is recomputed in f64.
// All sums are taken in a fixed order: no atomics.
#include "az_ops.hip.h"

namespace aznorm {

using namespace azops;

constexpr int NT = 256, MAX_C = 16384, MAX_G = 1024;

struct Args {
  const void *x, *r, *dy, *w, *b;
  void *y, *dx, *dr, *dw, *db;
  double *stats;   // [n][g]: mean, rstd
  double *part;    // forward, a sample in chunks: [n][chunk][g] sum, sum of squares
  float *cpart;    // backward, a sample in chunks: [n][chunk][c] sum dz, sum dz xhat
  float *csum;     // backward: [n][c] the same over the sample
  float *gsum;     // backward, a sample in chunks: [n][g] mean of dz w, mean of dz w xhat
  double *wpart;   // backward: [split][c] the channel sums of a share of the samples
  int64_t n;
  int hw, c, g, cg, chunks, per_chunk, act, param_f32, splits, cols, slices;
  double eps;
};

template <class T, int V> struct alignas(sizeof(T) * V) Vec { T v[V]; };
template <class T, int V> __device__ __forceinline__ void load(float *o, const T *p) {
  const Vec<T, V> t = *(const Vec<T, V> *)p;
#pragma unroll
  for (int j = 0; j < V; ++j) o[j] = to_f32(t.v[j]);
}
template <class T, int V> __device__ __forceinline__ void store(T *p, const float *o) {
  Vec<T, V> t;
#pragma unroll
  for (int j = 0; j < V; ++j) from_f32(o[j], t.v[j]);
  *(Vec<T, V> *)p = t;
}
// what a group's sums are taken about: its first value in sample x
template <class T> __device__ __forceinline__ double pivot_of(const T *x, int g, int cg) { return to_f32(x[g * cg]); }
template <class T> __device__ __forceinline__ float param(const void *p, int f32, int i, float none) {
  return p == nullptr ? none : f32 ? ((const float *)p)[i] : to_f32(((const T *)p)[i]);
}
// V neighbouring ones at once (the pointer is aligned to its elements only)
template <class T, int V> __device__ __forceinline__ void params(const void *p, int f32, int i, float none, float *o) {
  if (p == nullptr) {
#pragma unroll
    for (int j = 0; j < V; ++j) o[j] = none;
  } else if (f32) {
    __builtin_memcpy(o, (const float *)p + i, V * 4);
  } else {
    T t[V];
    __builtin_memcpy(t, (const T *)p + i, sizeof(t));
#pragma unroll
    for (int j = 0; j < V; ++j) o[j] = to_f32(t[j]);
  }
}
template <class T> __device__ __forceinline__ void put_param(void *p, int f32, int i, double v) {
  if (p == nullptr) return;
  if (f32) ((float *)p)[i] = (float)v;
  else from_f32((float)v, ((T *)p)[i]);
}

// of one group, as the elementwise part uses it: xhat = (x - mean) rstd with the mean as a pair of f32, (x - mh) rs + off
struct Stat {
  float mh, off, rs;
  __device__ __forceinline__ float xhat(float x) const { return fmaf(x - mh, rs, off); }
};
__device__ __forceinline__ Stat stat_of(double mean, double rstd) {
  const float mh = (float)mean;
  return Stat{mh, (float)(((double)mh - mean) * rstd), (float)rstd};
}

// 1 / (1 + 2^(-z log2 e)): off by |z| 2^-23 of itself at most where it is small, which z sigmoid(z) and the gradient share
__device__ __forceinline__ float sigmoid(float z) { return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * -1.44269504f)); }

// the activation of V values; `act` is uniform, so this is one branch for all of them
template <int V> __device__ __forceinline__ void act_fwd(float *z, int act) {
  if (act == AZ_ACT_RELU) {
#pragma unroll
    for (int j = 0; j < V; ++j) z[j] = z[j] > 0.0f || z[j] != z[j] ? z[j] : 0.0f;
  } else if (act == AZ_ACT_SILU) {
#pragma unroll
    for (int j = 0; j < V; ++j) z[j] *= sigmoid(z[j]);
  }
}

// V elements of a channel block: x, dy (and r) -> xhat and dz = dy act'(z).  z next to 0 (closer than f32 resolves z's terms) under
// relu: the sign from f64
template <int V, bool RES> __device__ __forceinline__ void grad(const float *x, const float *r, const float *w, const float *b, const Stat &st,
                                                                const double *sd, int act, float *d, float *xh) {
#pragma unroll
  for (int j = 0; j < V; ++j) xh[j] = st.xhat(x[j]);
  if (act == AZ_ACT_RELU) {
    float z[V];
    bool unsure = false;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float t = xh[j] * w[j], rj = RES ? r[j] : 0.0f;
      z[j] = (t + b[j]) + rj;
      unsure |= fabsf(z[j]) <= 0x1p-18f * (fabsf(t) + fabsf(b[j]) + fabsf(rj));
    }
    if (__builtin_expect(unsure, 0)) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        float wj = w[j], bj = b[j];
        asm volatile("" : "+v"(wj), "+v"(bj));  // (widened here, not ahead of the branch for every element)
        z[j] = fma(((double)x[j] - sd[0]) * sd[1], (double)wj, (double)bj) + (double)(RES ? r[j] : 0.0f) > 0.0 ? 1.0f : 0.0f;
      }
    }
#pragma unroll
    for (int j = 0; j < V; ++j) d[j] = z[j] > 0.0f ? d[j] : 0.0f;
  } else if (act == AZ_ACT_SILU) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float z = fmaf(xh[j], w[j], b[j]) + (RES ? r[j] : 0.0f), s = sigmoid(z);
      d[j] *= s * fmaf(z, 1.0f - s, 1.0f);
    }
  }
}

// How a workgroup walks pixels [p0, p1) of a sample: a pixel is CV = C / V vectors, TX threads side by side take them (looping when
// there are more), TY pixels at a time.  V never straddles a group (C / G is a multiple of it).
struct Walk {
  int cv, tx_n, ty_n, tx, ty;
  __device__ __forceinline__ Walk(int c, int v) {
    cv = c / v;
    tx_n = cv < NT ? cv : NT;
    ty_n = NT / tx_n;
    tx = threadIdx.x % tx_n;
    ty = threadIdx.x / tx_n;
  }
};

template <class T, int V> __global__ __launch_bounds__(NT) void k_gn_stats(Args a) {
  __shared__ double s_[NT], q_[NT], gs[MAX_G], gq[MAX_G];
  const int chunk = blockIdx.x % a.chunks, tid = threadIdx.x;
  const int64_t n = blockIdx.x / a.chunks;
  const Walk k(a.c, V);
  const int p0 = chunk * a.per_chunk, p1 = min(p0 + a.per_chunk, a.hw);
  const T *x = (const T *)a.x + n * a.hw * a.c;
  for (int g = tid; g < a.g; g += NT) gs[g] = gq[g] = 0.0;
  __syncthreads();
  const int cols_per_group = a.cg / V;
  for (int c0 = 0; c0 < k.cv; c0 += k.tx_n) {
    const int col = c0 + k.tx;
    double s = 0.0, q = 0.0;
    if (col < k.cv && k.ty < k.ty_n) {
      const double pivot = pivot_of(x, col * V / a.cg, a.cg);
#pragma unroll 4
      for (int p = p0 + k.ty; p < p1; p += k.ty_n) {
        float v[V];
        load<T, V>(v, x + (int64_t)p * a.c + col * V);
#pragma unroll
        for (int j = 0; j < V; ++j) { const double d = v[j] - pivot; s += d; q = fma(d, d, q); }
      }
    }
    s_[tid] = s;
    q_[tid] = q;
    __syncthreads();
    for (int g = tid; g < a.g; g += NT) {
      const int lo = max(g * cols_per_group, c0), hi = min((g + 1) * cols_per_group, min(c0 + k.tx_n, k.cv));
      for (int ty = 0; ty < k.ty_n; ++ty)
        for (int cc = lo; cc < hi; ++cc) { gs[g] += s_[ty * k.tx_n + cc - c0]; gq[g] += q_[ty * k.tx_n + cc - c0]; }
    }
    __syncthreads();
  }
  for (int g = tid; g < a.g; g += NT) {
    double *o = a.part + ((n * a.chunks + chunk) * a.g + g) * 2;
    o[0] = gs[g];
    o[1] = gq[g];
  }
}

// mean and 1 / sqrt(var + eps) of m values whose differences from the pivot have the sum s and the sum of squares q
__device__ __forceinline__ void finish(double s, double q, double m, double pivot, double eps, double &mean, double &rstd) {
  const double off = s / m;
  mean = pivot + off;
  // a group that holds an infinity or a NaN has no variance (fmax would hide it)
  rstd = q < 1e300 ? 1.0 / sqrt(fmax(q / m - off * off, 0.0) + eps) : NAN;
}

// the chunks' sums -> the statistics: one wave a (sample, group)
template <class T> __global__ __launch_bounds__(NT) void k_gn_stats_join(Args a) {
  const int64_t ng = blockIdx.x * (int64_t)(NT / 64) + (threadIdx.x >> 6), n = ng / a.g;
  const int g = (int)(ng - n * a.g), lane = threadIdx.x & 63;
  if (n >= a.n) return;
  double s = 0.0, q = 0.0;
#pragma unroll 4
  for (int i = lane; i < a.chunks; i += 64) { const double *p = a.part + ((n * a.chunks + i) * a.g + g) * 2; s += p[0]; q += p[1]; }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) { s += __shfl_xor(s, o); q += __shfl_xor(q, o); }
  if (lane == 0) finish(s, q, (double)a.hw * a.cg, pivot_of((const T *)a.x + n * a.hw * a.c, g, a.cg), a.eps, a.stats[ng * 2], a.stats[ng * 2 + 1]);
}

template <class T, int V> __global__ __launch_bounds__(NT) void k_gn_apply(Args a) {
  const int chunk = blockIdx.x % a.chunks;
  const int64_t n = blockIdx.x / a.chunks;
  const Walk k(a.c, V);
  const int p0 = chunk * a.per_chunk, p1 = min(p0 + a.per_chunk, a.hw);
  if (k.ty >= k.ty_n) return;
  const int64_t base = n * a.hw * a.c;
  for (int col = k.tx; col < k.cv; col += k.tx_n) {
    const double *sd = a.stats + (n * a.g + col * V / a.cg) * 2;
    const Stat s = stat_of(sd[0], sd[1]);
    float w[V], b[V];
    params<T, V>(a.w, a.param_f32, col * V, 1.0f, w);
    params<T, V>(a.b, a.param_f32, col * V, 0.0f, b);
#pragma unroll 2
    for (int p = p0 + k.ty; p < p1; p += k.ty_n) {
      const int64_t at = base + (int64_t)p * a.c + col * V;
      float v[V], r[V] = {};
      load<T, V>(v, (const T *)a.x + at);
      if (a.r) load<T, V>(r, (const T *)a.r + at);
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = fmaf(s.xhat(v[j]), w[j], b[j]) + r[j];
      act_fwd<V>(v, a.act);
      store<T, V>((T *)a.y + at, v);
    }
  }
}

// A thread's terms are summed in f32 over RUN pixels at most (off by RUN 2^-24 of their magnitudes) and the runs in f64: a thread may have any
// number of pixels.  The f64 sums lie in LDS from the start (in registers, 154 of them leave three waves a SIMD: 30.8 us for
// 4 x 512 x 128 x 127 f16 instead of 26).
constexpr int RUN = 64;
template <class T, int V> __global__ __launch_bounds__(NT) void k_gn_bwd_sums(Args a) {
  __shared__ double s_[NT * V], q_[NT * V];
  const int chunk = blockIdx.x % a.chunks, tid = threadIdx.x;
  const int64_t n = blockIdx.x / a.chunks, base = n * a.hw * a.c;
  const Walk k(a.c, V);
  const int p0 = chunk * a.per_chunk, p1 = min(p0 + a.per_chunk, a.hw);
  for (int c0 = 0; c0 < k.cv; c0 += k.tx_n) {
    const int col = c0 + k.tx;
#pragma unroll
    for (int j = 0; j < V; ++j) s_[j * NT + tid] = q_[j * NT + tid] = 0.0;
    if (col < k.cv && k.ty < k.ty_n) {
      const double *sd = a.stats + (n * a.g + col * V / a.cg) * 2;
      const double sd2[2] = {sd[0], sd[1]};
      const Stat st = stat_of(sd2[0], sd2[1]);
      float w[V], b[V];
      params<T, V>(a.w, a.param_f32, col * V, 1.0f, w);
      params<T, V>(a.b, a.param_f32, col * V, 0.0f, b);
      for (int p = p0 + k.ty; p < p1;) {
        const int end = min(p1 - p, RUN * k.ty_n) + p;
        float s[V] = {}, q[V] = {};
#pragma unroll 2
        for (; p < end; p += k.ty_n) {
          const int64_t at = base + (int64_t)p * a.c + col * V;
          float x[V], r[V] = {}, d[V];
          load<T, V>(x, (const T *)a.x + at);
          load<T, V>(d, (const T *)a.dy + at);
          if (a.r) load<T, V>(r, (const T *)a.r + at);
          float xh[V];
          grad<V, true>(x, r, w, b, st, sd2, a.act, d, xh);
#pragma unroll
          for (int j = 0; j < V; ++j) {
            s[j] += d[j];
            q[j] = fmaf(d[j], xh[j], q[j]);
          }
        }
#pragma unroll
        for (int j = 0; j < V; ++j) { s_[j * NT + tid] += s[j]; q_[j * NT + tid] += q[j]; }
      }
    }
    __syncthreads();
    const int cols = min(k.tx_n, k.cv - c0) * V;
    for (int e = tid; e < cols; e += NT) {
      double s = 0.0, q = 0.0;
      for (int ty = 0; ty < k.ty_n; ++ty) { const int t = e % V * NT + ty * k.tx_n + e / V; s += s_[t]; q += q_[t]; }
      float *o = a.cpart + ((n * a.chunks + chunk) * a.c + c0 * V + e) * 2;
      o[0] = (float)s;
      o[1] = (float)q;
    }
    __syncthreads();
  }
}

// the chunks' channel sums -> the sample's, and the two means a group's dx needs: one workgroup a (sample, group)
template <class T> __global__ __launch_bounds__(NT) void k_gn_bwd_join(Args a) {
  __shared__ double s_[NT], q_[NT], gs[NT / 64], gq[NT / 64];
  const int64_t n = blockIdx.x / a.g;
  const int g = (int)(blockIdx.x - n * a.g), tid = threadIdx.x;
  const int tx_n = a.cg < NT ? a.cg : NT, ty_n = NT / tx_n, tx = tid % tx_n, ty = tid / tx_n;
  double s1 = 0.0, q1 = 0.0;  // this thread's share of the group's weighted sums
  for (int c0 = 0; c0 < a.cg; c0 += tx_n) {
    const int c = g * a.cg + c0 + tx;
    double s = 0.0, q = 0.0;
    if (c0 + tx < a.cg && ty < ty_n)
#pragma unroll 8
      for (int i = ty; i < a.chunks; i += ty_n) { const float *p = a.cpart + ((n * a.chunks + i) * a.c + c) * 2; s += p[0]; q += p[1]; }
    s_[tid] = s;
    q_[tid] = q;
    __syncthreads();
    if (ty == 0 && c0 + tx < a.cg) {
      for (int y = 1; y < ty_n; ++y) { s += s_[y * tx_n + tx]; q += q_[y * tx_n + tx]; }
      a.csum[(n * a.c + c) * 2] = (float)s;
      a.csum[(n * a.c + c) * 2 + 1] = (float)q;
      const double w = param<T>(a.w, a.param_f32, c, 1.0f);
      s1 = fma(w, s, s1);
      q1 = fma(w, q, q1);
    }
    __syncthreads();
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) { s1 += __shfl_xor(s1, o); q1 += __shfl_xor(q1, o); }
  if ((tid & 63) == 0) { gs[tid >> 6] = s1; gq[tid >> 6] = q1; }
  __syncthreads();
  if (tid == 0) {
    const double m = (double)a.hw * a.cg;
    a.gsum[(n * a.g + g) * 2] = (float)((((gs[0] + gs[1]) + gs[2]) + gs[3]) / m);
    a.gsum[(n * a.g + g) * 2 + 1] = (float)((((gq[0] + gq[1]) + gq[2]) + gq[3]) / m);
  }
}

template <class T, int V> __global__ __launch_bounds__(NT) void k_gn_bwd_dx(Args a) {
  const int chunk = blockIdx.x % a.chunks;
  const int64_t n = blockIdx.x / a.chunks, base = n * a.hw * a.c;
  const Walk k(a.c, V);
  const int p0 = chunk * a.per_chunk, p1 = min(p0 + a.per_chunk, a.hw);
  if (k.ty >= k.ty_n) return;
  for (int col = k.tx; col < k.cv; col += k.tx_n) {
    const int g = col * V / a.cg;
    const double *sd = a.stats + (n * a.g + g) * 2;
    const double sd2[2] = {sd[0], sd[1]};
    const Stat st = stat_of(sd2[0], sd2[1]);
    const float m1 = a.gsum[(n * a.g + g) * 2], m2 = a.gsum[(n * a.g + g) * 2 + 1];
    float w[V], b[V];
    params<T, V>(a.w, a.param_f32, col * V, 1.0f, w);
    params<T, V>(a.b, a.param_f32, col * V, 0.0f, b);
#pragma unroll 2
    for (int p = p0 + k.ty; p < p1; p += k.ty_n) {
      const int64_t at = base + (int64_t)p * a.c + col * V;
      float x[V], r[V] = {}, d[V];
      load<T, V>(x, (const T *)a.x + at);
      load<T, V>(d, (const T *)a.dy + at);
      if (a.r) load<T, V>(r, (const T *)a.r + at);
      float xh[V];
      grad<V, true>(x, r, w, b, st, sd2, a.act, d, xh);
#pragma unroll
      for (int j = 0; j < V; ++j) x[j] = st.rs * (fmaf(d[j], w[j], -m1) - xh[j] * m2);
      if (a.dx) store<T, V>((T *)a.dx + at, x);
      if (a.dr) store<T, V>((T *)a.dr + at, d);
    }
  }
}

// A sample's channels fit a workgroup's registers: one workgroup takes `cols` vectors (whole groups, 64 lanes at most) of every pixel
// of a sample, so x is read once.  Its lanes keep their column for all pixels: weights, statistics and channel sums stay in registers.
// `cols` and the vectors of a group are powers of two: lanes of one group differ in the bits below `cgv` and from `cols` on.
template <class T> __device__ __forceinline__ void unpack(const u32x4 &w, float *o) {
  constexpr int N = Word<T>::N;
#pragma unroll
  for (int j = 0; j < 4 * N; ++j) o[j] = Word<T>::get(w[j / N], j % N);
}
template <class T> __device__ __forceinline__ u32x4 pack(const float *o) {
  constexpr int N = Word<T>::N;
  return u32x4{Word<T>::put(o), Word<T>::put(o + N), Word<T>::put(o + 2 * N), Word<T>::put(o + 3 * N)};
}

// the packed words are what lives from the first use to the second: without this the compiler keeps the unpacked values too (240
// registers instead of 100)
__device__ __forceinline__ void packed_only(u32x4 &w) { asm volatile("" : "+v"(w)); }

template <class T, int NV, bool RES> __global__ __launch_bounds__(NT) void k_gn_fwd_one(Args a) {
  constexpr int V = 16 / sizeof(T);
  __shared__ double part[NT / 64][64][2];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, cols = a.cols, cgv = a.cg / V;
  const int64_t n = blockIdx.x / a.slices;
  const int col = (int)(blockIdx.x - n * a.slices) * cols + (tid & (cols - 1)), cv = a.c / V, p0 = tid / cols, step = NT / cols;
  // the sample's bytes: a uniform base and a 32-bit offset (a resident sample has at most 1,024 pixels of 64 KiB).  Pixels behind the
  // sample read its last one, and do not count
  const int64_t base = n * a.hw * a.c * (int64_t)sizeof(T);
  const char *x = (const char *)a.x + base, *r = (const char *)a.r + base;
  auto at = [&](int i) { return (uint32_t)(min(p0 + i * step, a.hw - 1) * cv + col) * 16u; };
  u32x4 v[NV], rv[RES ? NV : 1];
#pragma unroll
  for (int i = 0; i < NV; ++i) v[i] = *(const u32x4 *)(x + at(i));
  if (RES) {
#pragma unroll
    for (int i = 0; i < NV; ++i) rv[i] = *(const u32x4 *)(r + at(i));
  }
  const int g = col / cgv;
  const double pivot = pivot_of((const T *)x, g, a.cg);
  double s = 0.0, q = 0.0;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if (p0 + i * step < a.hw) {
      float f[V];
      unpack<T>(v[i], f);
#pragma unroll
      for (int j = 0; j < V; ++j) { const double d = f[j] - pivot; s += d; q = fma(d, d, q); }
    }
    packed_only(v[i]);
  }
  for (int o = 1; o < 64; o <<= 1)
    if (o < cgv || o >= cols) { s += __shfl_xor(s, o); q += __shfl_xor(q, o); }
  const int gl = (tid & (cols - 1)) / cgv;
  if ((lane & (cgv - 1)) == 0 && lane < cols) { part[wave][gl][0] = s; part[wave][gl][1] = q; }
  float w[V], b[V];
#pragma unroll
  for (int j = 0; j < V; ++j) { w[j] = param<T>(a.w, a.param_f32, col * V + j, 1.0f); b[j] = param<T>(a.b, a.param_f32, col * V + j, 0.0f); }
  __syncthreads();
  s = ((part[0][gl][0] + part[1][gl][0]) + part[2][gl][0]) + part[3][gl][0];
  q = ((part[0][gl][1] + part[1][gl][1]) + part[2][gl][1]) + part[3][gl][1];
  double mean, rstd;
  finish(s, q, (double)a.hw * a.cg, pivot, a.eps, mean, rstd);
  if (tid < cols && (tid & (cgv - 1)) == 0) { a.stats[(n * a.g + g) * 2] = mean; a.stats[(n * a.g + g) * 2 + 1] = rstd; }
  const Stat st = stat_of(mean, rstd);
  char *y = (char *)a.y + base;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    float f[V], rf[V];
    unpack<T>(v[i], f);
    if (RES) unpack<T>(rv[i], rf);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      f[j] = fmaf(st.xhat(f[j]), w[j], b[j]);
      if (RES) f[j] += rf[j];
    }
    act_fwd<V>(f, a.act);
    const u32x4 o = pack<T>(f);
    if (p0 + i * step < a.hw) *(u32x4 *)(y + at(i)) = o;
  }
}

// the same for the gradient: x and dy are read once.  relu's dz is dy or 0, so it takes dy's place in its own type; silu's is computed
// again for dx (its residual, if any, is then read again).
template <class T, int NV, bool RES, int ACT> __global__ __launch_bounds__(NT) void k_gn_bwd_one(Args a) {
  constexpr int V = 16 / sizeof(T);
  __shared__ float part[NT / 64][64 * V][2];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, cols = a.cols, cgv = a.cg / V;
  const int64_t n = blockIdx.x / a.slices;
  const int lc = tid & (cols - 1), col = (int)(blockIdx.x - n * a.slices) * cols + lc, cv = a.c / V, p0 = tid / cols, step = NT / cols;
  const int64_t base = n * a.hw * a.c * (int64_t)sizeof(T);
  const char *x = (const char *)a.x + base, *r = (const char *)a.r + base, *dy = (const char *)a.dy + base;
  auto at = [&](int i) { return (uint32_t)(min(p0 + i * step, a.hw - 1) * cv + col) * 16u; };
  u32x4 xv[NV], dv[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    xv[i] = *(const u32x4 *)(x + at(i));
    dv[i] = *(const u32x4 *)(dy + at(i));
  }
  const int g = col / cgv;
  const double sd[2] = {a.stats[(n * a.g + g) * 2], a.stats[(n * a.g + g) * 2 + 1]};
  const Stat st = stat_of(sd[0], sd[1]);
  float w[V], b[V], s[V] = {}, q[V] = {};
#pragma unroll
  for (int j = 0; j < V; ++j) { w[j] = param<T>(a.w, a.param_f32, col * V + j, 1.0f); b[j] = param<T>(a.b, a.param_f32, col * V + j, 0.0f); }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const bool in = p0 + i * step < a.hw;
    float xf[V], rf[V], d[V], xh[V];
    if (RES) unpack<T>(*(const u32x4 *)(r + at(i)), rf);
    if (!in) dv[i] = u32x4{};
    unpack<T>(xv[i], xf);
    unpack<T>(dv[i], d);
    grad<V, RES>(xf, rf, w, b, st, sd, ACT, d, xh);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      s[j] += d[j];
      q[j] = fmaf(d[j], xh[j], q[j]);
      asm volatile("" : "+v"(s[j]), "+v"(q[j]));  // (or the sums are put off until the last vector, and every d and xhat is kept)
    }
    if (ACT == AZ_ACT_RELU) dv[i] = pack<T>(d);  // (exact)
    packed_only(xv[i]);
    packed_only(dv[i]);
  }
  for (int o = cols; o < 64; o <<= 1) {
#pragma unroll
    for (int j = 0; j < V; ++j) { s[j] += __shfl_xor(s[j], o); q[j] += __shfl_xor(q[j], o); }
  }
  if (lane < cols) {
#pragma unroll
    for (int j = 0; j < V; ++j) { part[wave][lc * V + j][0] = s[j]; part[wave][lc * V + j][1] = q[j]; }
  }
  __syncthreads();
  float m1 = 0.0f, m2 = 0.0f;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int e = lc * V + j;
    s[j] = ((part[0][e][0] + part[1][e][0]) + part[2][e][0]) + part[3][e][0];
    q[j] = ((part[0][e][1] + part[1][e][1]) + part[2][e][1]) + part[3][e][1];
    m1 = fmaf(w[j], s[j], m1);
    m2 = fmaf(w[j], q[j], m2);
    if (tid < cols) { a.csum[(n * a.c + col * V + j) * 2] = s[j]; a.csum[(n * a.c + col * V + j) * 2 + 1] = q[j]; }
  }
  if (a.dx == nullptr && a.dr == nullptr) return;
  for (int o = 1; o < cgv; o <<= 1) { m1 += __shfl_xor(m1, o); m2 += __shfl_xor(m2, o); }
  const float inv = 1.0f / ((float)a.hw * (float)a.cg);
  m1 *= inv;
  m2 *= inv;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const bool in = p0 + i * step < a.hw;
    float xf[V], rf[V], d[V], xh[V];
    unpack<T>(xv[i], xf);
    unpack<T>(dv[i], d);
    if (ACT == AZ_ACT_SILU) {
      if (RES) unpack<T>(*(const u32x4 *)(r + at(i)), rf);
      grad<V, RES>(xf, rf, w, b, st, sd, ACT, d, xh);
      dv[i] = pack<T>(d);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) xh[j] = st.xhat(xf[j]);
    }
#pragma unroll
    for (int j = 0; j < V; ++j) xf[j] = st.rs * (fmaf(d[j], w[j], -m1) - xh[j] * m2);
    const u32x4 o = pack<T>(xf);
    if (in && a.dx) *(u32x4 *)((char *)a.dx + base + at(i)) = o;
    if (in && a.dr) *(u32x4 *)((char *)a.dr + base + at(i)) = dv[i];
  }
}

// the samples' channel sums -> dweight, dbias: 4 channels (32 bytes of a row) x 256 rows at a time a workgroup.  Beyond 4,096 samples in
// `splits` shares (LAST false: into wpart), joined by a second pass.
constexpr int WB_C = 4, WB_NT = 1024;
template <class T, bool LAST> __global__ __launch_bounds__(WB_NT) void k_gn_wb(Args a) {
  __shared__ double s_[WB_NT / 64][WB_C], q_[WB_NT / 64][WB_C];
  const int tid = threadIdx.x, c = blockIdx.x * WB_C + tid % WB_C, lane = tid / WB_C;
  const bool joined = LAST && a.splits > 1;
  const int64_t rows = joined ? a.splits : a.n, per = LAST ? rows : (rows + a.splits - 1) / a.splits;
  const int64_t r0 = blockIdx.y * per, r1 = r0 + per < rows ? r0 + per : rows;
  double s = 0.0, q = 0.0;
  if (c < a.c) {
    if (joined) for (int64_t r = r0 + lane; r < r1; r += WB_NT / WB_C) { const double *p = a.wpart + (r * a.c + c) * 2; s += p[0]; q += p[1]; }
    else {
#pragma unroll 4
      for (int64_t r = r0 + lane; r < r1; r += WB_NT / WB_C) { const float2 p = *(const float2 *)(a.csum + (r * a.c + c) * 2); s += p.x; q += p.y; }
    }
  }
  for (int o = WB_C; o < 64; o <<= 1) { s += __shfl_xor(s, o); q += __shfl_xor(q, o); }
  if ((tid & 63) < WB_C) { s_[tid >> 6][tid % WB_C] = s; q_[tid >> 6][tid % WB_C] = q; }
  __syncthreads();
  if (tid >= WB_C || c >= a.c) return;
  s = q = 0.0;
  for (int w = 0; w < WB_NT / 64; ++w) { s += s_[w][tid]; q += q_[w][tid]; }
  if (LAST) {
    put_param<T>(a.db, a.param_f32, c, s);
    put_param<T>(a.dw, a.param_f32, c, q);
  } else {
    double *o = a.wpart + ((int64_t)blockIdx.y * a.c + c) * 2;
    o[0] = s;
    o[1] = q;
  }
}

// pixels of a sample are shared out so that there are workgroups enough (four a CU; two or three are slower, 4 x 512 x 128 x 127: 119 and 112 us
// against 109; eight are no faster and leave twice the partial sums to join), but never fewer than 32 pixels to one
static int chunks_of(int64_t n, int hw) {
  int64_t want = (1024 + n - 1) / n, most = (hw + 31) / 32;
  return (int)(want < 1 ? 1 : want < most ? want : most);
}
static int splits_of(int64_t n) { return n <= 4096 ? 1 : n < 65536 ? (int)(n / 1024) : 64; }

// doubles and floats of the workspace in this order: part | cpart, csum, gsum, wpart
static int64_t ws_forward(int64_t n, int hw, int g) { return n * chunks_of(n, hw) * g * 16; }
static int64_t up16(int64_t v) { return (v + 15) / 16 * 16; }
static int64_t ws_backward(int64_t n, int hw, int c, int g) {
  return up16(n * chunks_of(n, hw) * c * 8) + up16(n * c * 8) + up16(n * g * 8) + (int64_t)splits_of(n) * c * 16;
}

static int check(const char *&msg, int32_t dtype, int32_t param_dtype, int64_t n, int64_t hw, int32_t c, int32_t g, int32_t act, double eps) {
  if (dtype != AZ_NN_F32 && dtype != AZ_NN_BF16 && dtype != AZ_NN_F16) { msg = "group norm: unknown dtype"; return AZ_EINVAL; }
  if (param_dtype != AZ_NN_F32 && param_dtype != dtype) { msg = "group norm: weight and bias are f32 or of x's dtype"; return AZ_EINVAL; }
  if (act != AZ_ACT_NONE && act != AZ_ACT_RELU && act != AZ_ACT_SILU) { msg = "group norm: unknown activation"; return AZ_EINVAL; }
  if (n < 0 || hw < 0 || c < 1 || c > MAX_C || g < 1 || g > MAX_G || c % g) { msg = "group norm: 1 <= C <= 16,384 a multiple of the groups, at most 1,024 groups"; return AZ_EINVAL; }
  // (a workgroup of 256 a group, and a launch holds fewer than 2^32 threads)
  if (n >= (1 << 24) || hw > (1 << 28) || n * g >= (1 << 24)) { msg = "group norm: at most 2^24 - 1 groups in all samples, 2^28 pixels"; return AZ_EINVAL; }
  if (!(eps >= 0.0)) { msg = "group norm: eps >= 0"; return AZ_EINVAL; }
  return AZ_OK;
}

template <class F> static int by_type(int32_t dtype, int v, F f) {
  auto inner = [&](auto t) {
    using T = decltype(t);
    if constexpr (sizeof(T) == 2) { if (v == 8) return f(t, std::integral_constant<int, 8>{}); }
    return v >= 4 ? f(t, std::integral_constant<int, 4>{}) : v == 2 ? f(t, std::integral_constant<int, 2>{}) : f(t, std::integral_constant<int, 1>{});
  };
  return dtype == AZ_NN_F32 ? inner(float{}) : dtype == AZ_NN_BF16 ? inner(bf16_t{}) : inner(f16_t{});
}

// elements per load: up to 16 bytes, a divisor of a group's channels, and what every pointer is aligned to
static int vec_of(int32_t dtype, int cg, const void *const *ptrs, int np) {
  const int es = dtype == AZ_NN_F32 ? 4 : 2;
  int v = 16 / es;
  while (v > 1 && cg % v) v >>= 1;
  for (int i = 0; i < np; ++i)
    while (v > 1 && misaligned(ptrs[i], (uintptr_t)v * es)) v >>= 1;
  return v;
}

static int count_of(int need) { return need <= 4 ? need : need <= 6 ? 6 : need <= 8 ? 8 : need <= 12 ? 12 : 16; }  // (the vectors a thread holds)

// Columns of 16 bytes a workgroup takes where a sample's share fits its registers (nv vectors a thread), or 0: whole groups, a power
// of two, at least 64 bytes of a pixel side by side where the sample has them, and the fewest threads left idle.
static int cols_of(int32_t dtype, int v, int c, int cg, int hw, int max_nv, int &nv) {
  const int full = dtype == AZ_NN_F32 ? 4 : 8, cv = c / full, cgv = cg / full;
  if (v != full || (cgv & (cgv - 1))) return 0;
  int best = 0;
  double waste = 0.0;
  for (int cols = cgv > 4 ? cgv : 4; cols <= 64 && cv % cols == 0; cols *= 2) {
    const int need = (hw * (int64_t)cols + NT - 1) / NT <= max_nv ? (int)((hw * (int64_t)cols + NT - 1) / NT) : 0;
    if (need == 0) break;
    const int n = count_of(need);
    const double w = (double)n * NT / ((double)hw * cols) * (cols * 16 < 128 ? 1.1 : 1.0);
    if (best == 0 || w < waste) { best = cols; waste = w; nv = n; }
  }
  if (best == 0 && cv < 4 && (cv & (cv - 1)) == 0 && cgv <= cv) {  // (fewer than 64 bytes a pixel)
    const int64_t need = ((int64_t)hw * cv + NT - 1) / NT;
    if (need <= max_nv) {
      nv = count_of((int)need);
      best = cv;
    }
  }
  return best;
}

template <class F> static int by_count(int nv, F f) {
  switch (nv) {
    case 1: return f(std::integral_constant<int, 1>{});
    case 2: return f(std::integral_constant<int, 2>{});
    case 3: return f(std::integral_constant<int, 3>{});
    case 4: return f(std::integral_constant<int, 4>{});
    case 6: return f(std::integral_constant<int, 6>{});
    case 8: return f(std::integral_constant<int, 8>{});
    case 12: return f(std::integral_constant<int, 12>{});
    default: return f(std::integral_constant<int, 16>{});
  }
}
template <class F> static int by_dtype(int32_t dtype, F f) { return dtype == AZ_NN_F32 ? f(float{}) : dtype == AZ_NN_BF16 ? f(bf16_t{}) : f(f16_t{}); }

}  // namespace aznorm

extern "C" {

int64_t az_group_norm_workspace(int32_t backward, int64_t n, int64_t hw, int32_t c, int32_t groups) {
  using namespace aznorm;
  const char *msg = "";
  if (check(msg, AZ_NN_F32, AZ_NN_F32, n, hw, c, groups, AZ_ACT_NONE, 0.0) != AZ_OK) { fail(AZ_EINVAL, msg); return -1; }
  if (n == 0 || hw == 0) return 0;
  return backward ? ws_backward(n, (int)hw, c, groups) : ws_forward(n, (int)hw, groups);
}

int az_group_norm_forward(int32_t dtype, int32_t param_dtype, int64_t n, int64_t hw, int32_t c, int32_t groups, int32_t act, double eps,
                          const void *x_dev, const void *residual_dev, const void *weight_dev, const void *bias_dev, void *y_dev,
                          double *stats_dev, void *workspace_dev, int64_t workspace_bytes, void *stream) {
  using namespace aznorm;
  const char *msg = "";
  if (check(msg, dtype, param_dtype, n, hw, c, groups, act, eps) != AZ_OK) return fail(AZ_EINVAL, msg);
  if (n == 0 || hw == 0) return AZ_OK;
  const int es = dtype == AZ_NN_F32 ? 4 : 2, ps = param_dtype == AZ_NN_F32 ? 4 : 2;
  if (!x_dev || !y_dev || !stats_dev || !workspace_dev) return fail(AZ_EINVAL, "group norm: null argument");
  if (misaligned(x_dev, es) || misaligned(residual_dev, es) || misaligned(y_dev, es) || misaligned(weight_dev, ps) || misaligned(bias_dev, ps) ||
      misaligned(stats_dev, 8) || misaligned(workspace_dev, 16))
    return fail(AZ_EINVAL, "group norm: misaligned pointer");
  if (workspace_bytes < ws_forward(n, (int)hw, groups)) return fail(AZ_EINVAL, "group norm: workspace below az_group_norm_workspace()");
  hipStream_t s = (hipStream_t)stream;
  DeviceGuard guard(s);
  if (!guard.ok) return fail(AZ_EHIP, "group norm: cannot select the stream's device");
  Args a{};
  a.x = x_dev; a.r = residual_dev; a.w = weight_dev; a.b = bias_dev; a.y = y_dev;
  a.stats = stats_dev; a.part = (double *)workspace_dev;
  a.n = n; a.hw = (int)hw; a.c = c; a.g = groups; a.cg = c / groups; a.act = act; a.param_f32 = param_dtype == AZ_NN_F32; a.eps = eps;
  a.chunks = chunks_of(n, a.hw); a.per_chunk = (a.hw + a.chunks - 1) / a.chunks;
  const void *ptrs[] = {x_dev, residual_dev, y_dev};
  const int vec = vec_of(dtype, a.cg, ptrs, 3);
  int nv = 0;
  a.cols = cols_of(dtype, vec, c, a.cg, a.hw, 16, nv);
  if (a.cols) {
    a.slices = c / (16 / es) / a.cols;
    return by_dtype(dtype, [&](auto t) {
      return by_count(nv, [&](auto k) {
        using T = decltype(t);
        constexpr int NV = decltype(k)::value;
        const dim3 grid((unsigned)(n * a.slices));
        if (a.r) hipLaunchKernelGGL((k_gn_fwd_one<T, NV, true>), grid, dim3(NT), 0, s, a);
        else hipLaunchKernelGGL((k_gn_fwd_one<T, NV, false>), grid, dim3(NT), 0, s, a);
        return launched("k_gn_fwd_one");
      });
    });
  }
  return by_type(dtype, vec, [&](auto t, auto v) {
    using T = decltype(t);
    constexpr int V = decltype(v)::value;
    const dim3 grid((unsigned)(n * a.chunks));
    hipLaunchKernelGGL((k_gn_stats<T, V>), grid, dim3(NT), 0, s, a);
    hipLaunchKernelGGL(k_gn_stats_join<T>, dim3((unsigned)((n * groups + NT / 64 - 1) / (NT / 64))), dim3(NT), 0, s, a);
    hipLaunchKernelGGL((k_gn_apply<T, V>), grid, dim3(NT), 0, s, a);
    return launched("k_gn_forward");
  });
}

int az_group_norm_backward(int32_t dtype, int32_t param_dtype, int64_t n, int64_t hw, int32_t c, int32_t groups, int32_t act,
                           const void *x_dev, const void *residual_dev, const void *weight_dev, const void *bias_dev, const void *dy_dev,
                           const double *stats_dev, void *dx_dev, void *dresidual_dev, void *dweight_dev, void *dbias_dev,
                           void *workspace_dev, int64_t workspace_bytes, void *stream) {
  using namespace aznorm;
  const char *msg = "";
  if (check(msg, dtype, param_dtype, n, hw, c, groups, act, 0.0) != AZ_OK) return fail(AZ_EINVAL, msg);
  const bool empty = n == 0 || hw == 0;
  const int es = dtype == AZ_NN_F32 ? 4 : 2, ps = param_dtype == AZ_NN_F32 ? 4 : 2;
  if (!empty && (!x_dev || !dy_dev || !stats_dev || !workspace_dev)) return fail(AZ_EINVAL, "group norm: null argument");
  if (misaligned(x_dev, es) || misaligned(residual_dev, es) || misaligned(dy_dev, es) || misaligned(dx_dev, es) || misaligned(dresidual_dev, es) ||
      misaligned(weight_dev, ps) || misaligned(bias_dev, ps) || misaligned(dweight_dev, ps) || misaligned(dbias_dev, ps) || misaligned(stats_dev, 8) ||
      misaligned(workspace_dev, 16))
    return fail(AZ_EINVAL, "group norm: misaligned pointer");
  if (!empty && workspace_bytes < ws_backward(n, (int)hw, c, groups)) return fail(AZ_EINVAL, "group norm: workspace below az_group_norm_workspace()");
  hipStream_t s = (hipStream_t)stream;
  DeviceGuard guard(s);
  if (!guard.ok) return fail(AZ_EHIP, "group norm: cannot select the stream's device");
  Args a{};
  a.x = x_dev; a.r = residual_dev; a.w = weight_dev; a.b = bias_dev; a.dy = dy_dev; a.dx = dx_dev; a.dr = dresidual_dev; a.dw = dweight_dev; a.db = dbias_dev;
  a.stats = (double *)stats_dev;
  a.n = n; a.hw = (int)hw; a.c = c; a.g = groups; a.cg = c / groups; a.act = act; a.param_f32 = param_dtype == AZ_NN_F32;
  a.splits = splits_of(n);
  if (empty) {  // no samples: the parameters' gradients are zero
    a.n = 0;
    a.splits = 1;
    return by_dtype(dtype, [&](auto t) {
      hipLaunchKernelGGL((k_gn_wb<decltype(t), true>), dim3((c + WB_C - 1) / WB_C), dim3(WB_NT), 0, s, a);
      return launched("k_gn_wb");
    });
  }
  a.chunks = chunks_of(n, a.hw); a.per_chunk = (a.hw + a.chunks - 1) / a.chunks;
  char *ws = (char *)workspace_dev;
  a.cpart = (float *)ws;
  a.csum = (float *)(ws += up16(n * a.chunks * c * 8));
  a.gsum = (float *)(ws += up16(n * c * 8));
  a.wpart = (double *)(ws + up16(n * groups * 8));
  const bool params = dweight_dev || dbias_dev;
  const void *ptrs[] = {x_dev, residual_dev, dy_dev, dx_dev, dresidual_dev};
  const int vec = vec_of(dtype, a.cg, ptrs, 5);
  int nv = 0, rc;
  a.cols = cols_of(dtype, vec, c, a.cg, a.hw, 8, nv);
  if (a.cols) {
    a.slices = c / (16 / es) / a.cols;
    rc = by_dtype(dtype, [&](auto t) {
      return by_count(nv, [&](auto k) {
        using T = decltype(t);
        constexpr int NV = decltype(k)::value <= 8 ? decltype(k)::value : 8;
        const dim3 grid((unsigned)(n * a.slices));
        auto go = [&](auto act) {
          constexpr int ACT = decltype(act)::value;
          if (a.r) hipLaunchKernelGGL((k_gn_bwd_one<T, NV, true, ACT>), grid, dim3(NT), 0, s, a);
          else hipLaunchKernelGGL((k_gn_bwd_one<T, NV, false, ACT>), grid, dim3(NT), 0, s, a);
        };
        if (act == AZ_ACT_RELU) go(std::integral_constant<int, AZ_ACT_RELU>{});
        else if (act == AZ_ACT_SILU) go(std::integral_constant<int, AZ_ACT_SILU>{});
        else go(std::integral_constant<int, AZ_ACT_NONE>{});
        return launched("k_gn_bwd_one");
      });
    });
  } else {
    rc = by_type(dtype, vec, [&](auto t, auto v) {
      using T = decltype(t);
      constexpr int V = decltype(v)::value;
      const dim3 grid((unsigned)(n * a.chunks));
      hipLaunchKernelGGL((k_gn_bwd_sums<T, V>), grid, dim3(NT), 0, s, a);
      hipLaunchKernelGGL((k_gn_bwd_join<T>), dim3((unsigned)(n * groups)), dim3(NT), 0, s, a);
      if (dx_dev || dresidual_dev) hipLaunchKernelGGL((k_gn_bwd_dx<T, V>), grid, dim3(NT), 0, s, a);
      return launched("k_gn_backward");
    });
  }
  if (rc != AZ_OK || !params) return rc;
  return by_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    if (a.splits > 1) hipLaunchKernelGGL((k_gn_wb<T, false>), dim3((c + WB_C - 1) / WB_C, a.splits), dim3(WB_NT), 0, s, a);
    hipLaunchKernelGGL((k_gn_wb<T, true>), dim3((c + WB_C - 1) / WB_C), dim3(WB_NT), 0, s, a);
    return launched("k_gn_wb");
  });
}

}  // extern "C"
