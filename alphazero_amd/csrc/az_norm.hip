// az_norm.hip -- group norm with an activation over channels-last samples, forward and backward (gfx950).
//
//   a sample is (HW pixels, C channels), channels consecutive; group g = C / G consecutive channels of every pixel
//   xhat = (x - mean) rstd,  rstd = 1 / sqrt(var + eps),  z = xhat w + b (+ r),  y = act(z),  act: none, relu, silu
//   dz = dy act'(z);  dr = dz;  dw = sum dz xhat;  db = sum dz;
//   dx = rstd (dz w - mean_g(dz w) - xhat mean_g(dz w xhat))
//
// Bound by bytes: forward reads x (and r) and writes y, backward reads x, dy (and r) and writes dx (and dr).
// Mean and variance come from f64 sums of x and x^2 (the products of two f32 are exact in f64, so one pass is enough even where
// |mean| is 10^5 standard deviations); the mean is kept as a pair of f32 for the subtraction, everything per element is f32, and
// each output is rounded once.  A relu's gradient hangs on the sign of z: where f32 cannot tell it, z is recomputed in f64.
// All sums are taken in a fixed order: no atomics.
#include "az_ops.hip.h"

namespace aznorm {

using namespace azops;

constexpr int NT = 256, MAX_C = 16384, MAX_G = 1024;

struct Args {
  const void *x, *r, *dy, *w, *b;
  void *y, *dx, *dr, *dw, *db;
  double *stats;   // [n][g]: mean, rstd
  double *part;    // forward: [n][chunk][g] sum, sum of squares
  float *cpart;    // backward: [n][chunk][c] sum dz, sum dz xhat
  double *wpart;   // backward: [split][c] the same, over samples and chunks
  int n, hw, c, g, cg, chunks, per_chunk, act, param_f32, splits;
  float eps;
  int64_t rows;    // n * chunks
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
template <class T> __device__ __forceinline__ float param(const void *p, int f32, int i, float none) {
  return p == nullptr ? none : f32 ? ((const float *)p)[i] : to_f32(((const T *)p)[i]);
}
template <class T> __device__ __forceinline__ void put_param(void *p, int f32, int i, double v) {
  if (p == nullptr) return;
  if (f32) ((float *)p)[i] = (float)v;
  else from_f32((float)v, ((T *)p)[i]);
}

struct Stat {  // of one group, as the elementwise part uses it
  float mh, ml, rs;
};
__device__ __forceinline__ Stat stat_of(double mean, double rstd) {
  const float mh = (float)mean;
  return Stat{mh, (float)(mean - (double)mh), (float)rstd};
}

__device__ __forceinline__ float sigmoid(float z) { return __builtin_amdgcn_rcpf(1.0f + expf(-z)); }
__device__ __forceinline__ float act_fwd(float z, int act) { return act == AZ_ACT_RELU ? (z > 0.0f || z != z ? z : 0.0f) : act == AZ_ACT_SILU ? z * sigmoid(z) : z; }

// dy act'(z).  z next to 0 (closer than f32 resolves z's terms) under relu: the sign from f64
__device__ __forceinline__ float act_bwd(float dy, float z, float x, float xh, float w, float b, float r, int act, const double *st) {
  if (act == AZ_ACT_RELU) {
    bool on = z > 0.0f;
    if (__builtin_expect(fabsf(z) <= 0x1p-18f * (fabsf(xh * w) + fabsf(b) + fabsf(r)), 0))
      on = fma(((double)x - st[0]) * st[1], (double)w, (double)b) + (double)r > 0.0;
    return on ? dy : 0.0f;
  }
  if (act == AZ_ACT_SILU) {
    const float s = sigmoid(z);
    return dy * (s * fmaf(z, 1.0f - s, 1.0f));
  }
  return dy;
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
    if (col < k.cv && k.ty < k.ty_n)
      for (int p = p0 + k.ty; p < p1; p += k.ty_n) {
        float v[V];
        load<T, V>(v, x + (int64_t)p * a.c + col * V);
#pragma unroll
        for (int j = 0; j < V; ++j) { const double d = v[j]; s += d; q = fma(d, d, q); }
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

template <class T, int V> __global__ __launch_bounds__(NT) void k_gn_apply(Args a) {
  __shared__ Stat st[MAX_G];
  const int chunk = blockIdx.x % a.chunks, tid = threadIdx.x;
  const int64_t n = blockIdx.x / a.chunks;
  const double m = (double)a.hw * a.cg;
  for (int g = tid; g < a.g; g += NT) {
    double s = 0.0, q = 0.0;
    for (int i = 0; i < a.chunks; ++i) { const double *p = a.part + ((n * a.chunks + i) * a.g + g) * 2; s += p[0]; q += p[1]; }
    const double mean = s / m, var = fmax(q / m - mean * mean, 0.0), rstd = 1.0 / sqrt(var + (double)a.eps);
    const double rs = q < 1e300 ? rstd : NAN;  // a sample that holds an infinity or a NaN has no variance (fmax would hide it)
    st[g] = stat_of(mean, rs);
    if (chunk == 0) { a.stats[(n * a.g + g) * 2] = mean; a.stats[(n * a.g + g) * 2 + 1] = rs; }
  }
  __syncthreads();
  const Walk k(a.c, V);
  const int p0 = chunk * a.per_chunk, p1 = min(p0 + a.per_chunk, a.hw);
  if (k.ty >= k.ty_n) return;
  const int64_t base = n * a.hw * a.c;
  for (int col = k.tx; col < k.cv; col += k.tx_n) {
    const Stat s = st[col * V / a.cg];
    float w[V], b[V];
#pragma unroll
    for (int j = 0; j < V; ++j) { w[j] = param<T>(a.w, a.param_f32, col * V + j, 1.0f); b[j] = param<T>(a.b, a.param_f32, col * V + j, 0.0f); }
    for (int p = p0 + k.ty; p < p1; p += k.ty_n) {
      const int64_t at = base + (int64_t)p * a.c + col * V;
      float v[V], r[V] = {};
      load<T, V>(v, (const T *)a.x + at);
      if (a.r) load<T, V>(r, (const T *)a.r + at);
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = act_fwd(fmaf(((v[j] - s.mh) - s.ml) * s.rs, w[j], b[j]) + r[j], a.act);
      store<T, V>((T *)a.y + at, v);
    }
  }
}

template <class T, int V> __global__ __launch_bounds__(NT) void k_gn_bwd_sums(Args a) {
  __shared__ float s_[NT * V], q_[NT * V];
  const int chunk = blockIdx.x % a.chunks, tid = threadIdx.x;
  const int64_t n = blockIdx.x / a.chunks, base = n * a.hw * a.c;
  const Walk k(a.c, V);
  const int p0 = chunk * a.per_chunk, p1 = min(p0 + a.per_chunk, a.hw);
  for (int c0 = 0; c0 < k.cv; c0 += k.tx_n) {
    const int col = c0 + k.tx;
    float s[V] = {}, q[V] = {};
    if (col < k.cv && k.ty < k.ty_n) {
      const double *sd = a.stats + (n * a.g + col * V / a.cg) * 2;
      const double sd2[2] = {sd[0], sd[1]};
      const Stat st = stat_of(sd2[0], sd2[1]);
      float w[V], b[V];
#pragma unroll
      for (int j = 0; j < V; ++j) { w[j] = param<T>(a.w, a.param_f32, col * V + j, 1.0f); b[j] = param<T>(a.b, a.param_f32, col * V + j, 0.0f); }
      for (int p = p0 + k.ty; p < p1; p += k.ty_n) {
        const int64_t at = base + (int64_t)p * a.c + col * V;
        float x[V], r[V] = {}, d[V];
        load<T, V>(x, (const T *)a.x + at);
        load<T, V>(d, (const T *)a.dy + at);
        if (a.r) load<T, V>(r, (const T *)a.r + at);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float xh = ((x[j] - st.mh) - st.ml) * st.rs;
          const float dz = act_bwd(d[j], fmaf(xh, w[j], b[j]) + r[j], x[j], xh, w[j], b[j], r[j], a.act, sd2);
          s[j] += dz;
          q[j] = fmaf(dz, xh, q[j]);
        }
      }
    }
#pragma unroll
    for (int j = 0; j < V; ++j) { s_[tid * V + j] = s[j]; q_[tid * V + j] = q[j]; }
    __syncthreads();
    const int cols = min(k.tx_n, k.cv - c0) * V;
    for (int e = tid; e < cols; e += NT) {
      float ss = 0.0f, qq = 0.0f;
      for (int ty = 0; ty < k.ty_n; ++ty) { ss += s_[ty * k.tx_n * V + e]; qq += q_[ty * k.tx_n * V + e]; }
      float *o = a.cpart + ((n * a.chunks + chunk) * a.c + c0 * V + e) * 2;
      o[0] = ss;
      o[1] = qq;
    }
    __syncthreads();
  }
}

template <class T, int V> __global__ __launch_bounds__(NT) void k_gn_bwd_dx(Args a) {
  __shared__ float c1[MAX_G], c2[MAX_G];
  const int chunk = blockIdx.x % a.chunks, tid = threadIdx.x;
  const int64_t n = blockIdx.x / a.chunks, base = n * a.hw * a.c;
  const double m = (double)a.hw * a.cg;
  for (int g = tid; g < a.g; g += NT) {
    double s = 0.0, q = 0.0;
    for (int c = g * a.cg; c < (g + 1) * a.cg; ++c) {
      const double w = param<T>(a.w, a.param_f32, c, 1.0f);
      for (int i = 0; i < a.chunks; ++i) { const float *p = a.cpart + ((n * a.chunks + i) * a.c + c) * 2; s = fma(w, (double)p[0], s); q = fma(w, (double)p[1], q); }
    }
    c1[g] = (float)(s / m);
    c2[g] = (float)(q / m);
  }
  __syncthreads();
  const Walk k(a.c, V);
  const int p0 = chunk * a.per_chunk, p1 = min(p0 + a.per_chunk, a.hw);
  if (k.ty >= k.ty_n) return;
  for (int col = k.tx; col < k.cv; col += k.tx_n) {
    const int g = col * V / a.cg;
    const double *sd = a.stats + (n * a.g + g) * 2;
    const double sd2[2] = {sd[0], sd[1]};
    const Stat st = stat_of(sd2[0], sd2[1]);
    const float m1 = c1[g], m2 = c2[g];
    float w[V], b[V];
#pragma unroll
    for (int j = 0; j < V; ++j) { w[j] = param<T>(a.w, a.param_f32, col * V + j, 1.0f); b[j] = param<T>(a.b, a.param_f32, col * V + j, 0.0f); }
    for (int p = p0 + k.ty; p < p1; p += k.ty_n) {
      const int64_t at = base + (int64_t)p * a.c + col * V;
      float x[V], r[V] = {}, d[V];
      load<T, V>(x, (const T *)a.x + at);
      load<T, V>(d, (const T *)a.dy + at);
      if (a.r) load<T, V>(r, (const T *)a.r + at);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float xh = ((x[j] - st.mh) - st.ml) * st.rs;
        d[j] = act_bwd(d[j], fmaf(xh, w[j], b[j]) + r[j], x[j], xh, w[j], b[j], r[j], a.act, sd2);
        x[j] = st.rs * (fmaf(d[j], w[j], -m1) - xh * m2);
      }
      if (a.dx) store<T, V>((T *)a.dx + at, x);
      if (a.dr) store<T, V>((T *)a.dr + at, d);
    }
  }
}

// per-channel sums over samples and chunks: 64 channels x 4 row lanes a workgroup, `splits` shares of the rows, then one pass over those
template <class T> __global__ __launch_bounds__(NT) void k_gn_wb_part(Args a) {
  __shared__ double s_[NT], q_[NT];
  const int c = blockIdx.x * 64 + (threadIdx.x & 63), lane = threadIdx.x >> 6;
  const int64_t per = (a.rows + a.splits - 1) / a.splits, r0 = blockIdx.y * per, r1 = r0 + per < a.rows ? r0 + per : a.rows;
  double s = 0.0, q = 0.0;
  if (c < a.c)
    for (int64_t r = r0 + lane; r < r1; r += 4) { const float *p = a.cpart + (r * a.c + c) * 2; s += p[0]; q += p[1]; }
  s_[threadIdx.x] = s;
  q_[threadIdx.x] = q;
  __syncthreads();
  if (lane == 0 && c < a.c) {
    for (int l = 1; l < 4; ++l) { s += s_[l * 64 + threadIdx.x]; q += q_[l * 64 + threadIdx.x]; }
    double *o = a.wpart + ((int64_t)blockIdx.y * a.c + c) * 2;
    o[0] = s;
    o[1] = q;
  }
}
template <class T> __global__ __launch_bounds__(NT) void k_gn_wb(Args a) {
  const int c = blockIdx.x * NT + threadIdx.x;
  if (c >= a.c) return;
  double s = 0.0, q = 0.0;
  for (int i = 0; i < a.splits; ++i) { const double *p = a.wpart + ((int64_t)i * a.c + c) * 2; s += p[0]; q += p[1]; }
  put_param<T>(a.db, a.param_f32, c, s);
  put_param<T>(a.dw, a.param_f32, c, q);
}

// pixels of a sample are shared out so that there are workgroups enough, but never fewer than 32 pixels to one
static int chunks_of(int64_t n, int hw) {
  int64_t want = (2048 + n - 1) / n, most = (hw + 31) / 32;
  return (int)(want < 1 ? 1 : want < most ? want : most);
}
static int splits_of(int64_t rows) { return rows < 256 ? 1 : rows < 16384 ? (int)(rows / 256) + 1 : 64; }

static int64_t ws_forward(int64_t n, int hw, int g) { return n * chunks_of(n, hw) * g * 16; }
static int64_t ws_backward(int64_t n, int hw, int c) {
  const int64_t rows = n * chunks_of(n, hw);
  return rows * c * 8 + (int64_t)splits_of(rows) * c * 16;
}

static int check(const char *&msg, int32_t dtype, int32_t param_dtype, int64_t n, int64_t hw, int32_t c, int32_t g, int32_t act, double eps) {
  if (dtype != AZ_NN_F32 && dtype != AZ_NN_BF16 && dtype != AZ_NN_F16) { msg = "group norm: unknown dtype"; return AZ_EINVAL; }
  if (param_dtype != AZ_NN_F32 && param_dtype != dtype) { msg = "group norm: weight and bias are f32 or of x's dtype"; return AZ_EINVAL; }
  if (act != AZ_ACT_NONE && act != AZ_ACT_RELU && act != AZ_ACT_SILU) { msg = "group norm: unknown activation"; return AZ_EINVAL; }
  if (n < 0 || hw < 0 || c < 1 || c > MAX_C || g < 1 || g > MAX_G || c % g) { msg = "group norm: 1 <= C <= 16,384 a multiple of the groups, at most 1,024 groups"; return AZ_EINVAL; }
  if (n > (1 << 28) || hw > (1 << 28)) { msg = "group norm: at most 2^28 samples of 2^28 pixels"; return AZ_EINVAL; }
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

}  // namespace aznorm

extern "C" {

int64_t az_group_norm_workspace(int32_t backward, int64_t n, int64_t hw, int32_t c, int32_t groups) {
  using namespace aznorm;
  const char *msg = "";
  if (check(msg, AZ_NN_F32, AZ_NN_F32, n, hw, c, groups, AZ_ACT_NONE, 0.0) != AZ_OK) { fail(AZ_EINVAL, msg); return -1; }
  if (n == 0 || hw == 0) return 0;
  return backward ? ws_backward(n, (int)hw, c) : ws_forward(n, (int)hw, groups);
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
      misaligned(stats_dev, 8) || misaligned(workspace_dev, 8))
    return fail(AZ_EINVAL, "group norm: misaligned pointer");
  if (workspace_bytes < ws_forward(n, (int)hw, groups)) return fail(AZ_EINVAL, "group norm: workspace below az_group_norm_workspace()");
  hipStream_t s = (hipStream_t)stream;
  DeviceGuard guard(s);
  if (!guard.ok) return fail(AZ_EHIP, "group norm: cannot select the stream's device");
  Args a{};
  a.x = x_dev; a.r = residual_dev; a.w = weight_dev; a.b = bias_dev; a.y = y_dev;
  a.stats = stats_dev; a.part = (double *)workspace_dev;
  a.n = (int)n; a.hw = (int)hw; a.c = c; a.g = groups; a.cg = c / groups; a.act = act; a.param_f32 = param_dtype == AZ_NN_F32; a.eps = (float)eps;
  a.chunks = chunks_of(n, a.hw); a.per_chunk = (a.hw + a.chunks - 1) / a.chunks;
  const void *ptrs[] = {x_dev, residual_dev, y_dev};
  return by_type(dtype, vec_of(dtype, a.cg, ptrs, 3), [&](auto t, auto v) {
    using T = decltype(t);
    constexpr int V = decltype(v)::value;
    const dim3 grid((unsigned)(n * a.chunks));
    hipLaunchKernelGGL((k_gn_stats<T, V>), grid, dim3(NT), 0, s, a);
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
      misaligned(workspace_dev, 8))
    return fail(AZ_EINVAL, "group norm: misaligned pointer");
  if (!empty && workspace_bytes < ws_backward(n, (int)hw, c)) return fail(AZ_EINVAL, "group norm: workspace below az_group_norm_workspace()");
  hipStream_t s = (hipStream_t)stream;
  DeviceGuard guard(s);
  if (!guard.ok) return fail(AZ_EHIP, "group norm: cannot select the stream's device");
  Args a{};
  a.x = x_dev; a.r = residual_dev; a.w = weight_dev; a.b = bias_dev; a.dy = dy_dev; a.dx = dx_dev; a.dr = dresidual_dev; a.dw = dweight_dev; a.db = dbias_dev;
  a.stats = (double *)stats_dev;
  a.n = (int)n; a.hw = (int)hw; a.c = c; a.g = groups; a.cg = c / groups; a.act = act; a.param_f32 = param_dtype == AZ_NN_F32;
  if (empty) {  // no samples: the parameters' gradients are zero
    a.splits = 0;
    return by_type(dtype, 1, [&](auto t, auto) {
      hipLaunchKernelGGL((k_gn_wb<decltype(t)>), dim3((c + NT - 1) / NT), dim3(NT), 0, s, a);
      return launched("k_gn_wb");
    });
  }
  a.chunks = chunks_of(n, a.hw); a.per_chunk = (a.hw + a.chunks - 1) / a.chunks;
  a.rows = n * a.chunks; a.splits = splits_of(a.rows);
  a.cpart = (float *)workspace_dev; a.wpart = (double *)((char *)workspace_dev + a.rows * c * 8);
  const void *ptrs[] = {x_dev, residual_dev, dy_dev, dx_dev, dresidual_dev};
  return by_type(dtype, vec_of(dtype, a.cg, ptrs, 5), [&](auto t, auto v) {
    using T = decltype(t);
    constexpr int V = decltype(v)::value;
    const dim3 grid((unsigned)(n * a.chunks));
    hipLaunchKernelGGL((k_gn_bwd_sums<T, V>), grid, dim3(NT), 0, s, a);
    if (dx_dev || dresidual_dev) hipLaunchKernelGGL((k_gn_bwd_dx<T, V>), grid, dim3(NT), 0, s, a);
    if (dweight_dev || dbias_dev) {
      hipLaunchKernelGGL((k_gn_wb_part<T>), dim3((c + 63) / 64, a.splits), dim3(NT), 0, s, a);
      hipLaunchKernelGGL((k_gn_wb<T>), dim3((c + NT - 1) / NT), dim3(NT), 0, s, a);
    }
    return launched("k_gn_backward");
  });
}

}  // extern "C"
