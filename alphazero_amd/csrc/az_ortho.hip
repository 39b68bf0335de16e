// az_ortho.hip -- orthogonalising updates by Newton-Schulz products, a whole network's matrices per call (gfx950).
//
//   X0 = M / (|M|_F + eps), transposed if M has more rows than columns (S = short side, L = long side);
//   per step:  A = X X^T,   B = b A + c A^2,   X <- a X + B X
//
// All three are products of the form C[i][j] = sum_k P[i][k] Q[j][k] with k consecutive in both operands: A from X with itself, A^2
// from the symmetric A with itself, B X from B and the transpose of X, which every step writes beside X.  Of the symmetric results
// only the tiles on and above the diagonal are computed; the others are their mirror images.
//
// Arithmetic: f16 matrix instructions with f32 sums.  For f32 and f16 matrices an operand is a pair of f16, hi = f16(v) and
// lo = f16(v - hi), and a product is hi hi + hi lo + lo hi: 22 bits of each factor, three matrix instructions, several times the rate
// of the f32 ones.  For bf16 matrices hi alone holds more (11 bits) than the result will (8).  Stored values are scaled by powers of two
// (X: 2^12, A and B: 2^9) so that lo stays clear of f16's smallest steps; the host bounds the singular values (az_orthogonalize), so
// nothing overflows.  Buffers are zero padded to whole tiles and the padding stays zero: no product has a border case.
#include "az_ops.hip.h"

#include <cmath>

namespace azortho {

using namespace azops;

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int NT = 256, MAX_M = 64, NORM_PARTS = 64, TILE = 64, KS = 32, PITCH = KS + 8;
constexpr float SX = 4096.0f, SA = 512.0f;  // scales of the stored X and of the stored A and B

struct Mat {
  const void *in;
  void *out;
  uint64_t ws;  // byte offset of this matrix's buffers
  int32_t rows, cols;
};
struct Args {
  Mat m[MAX_M];
  char *ws;
  int32_t count, planes, cur;
  float a, b, c;
  double eps;
};

// one matrix's buffers in the workspace: norm parts (f64), then f16 planes (hi, lo): X [SP][LP], two X^T [LP][SP], A and B [SP][SP]
struct Lay {
  int s, l, sp, lp, planes;
  bool tall;
  __host__ __device__ Lay(int rows, int cols, int planes_) {
    tall = rows > cols;
    s = tall ? cols : rows;
    l = tall ? rows : cols;
    sp = (s + TILE - 1) / TILE * TILE;
    lp = (l + TILE - 1) / TILE * TILE;
    planes = planes_;
  }
  __host__ __device__ int64_t xn() const { return (int64_t)sp * lp; }
  __host__ __device__ int64_t an() const { return (int64_t)sp * sp; }
  __host__ __device__ int64_t x() const { return NORM_PARTS * 8; }
  __host__ __device__ int64_t xt(int which) const { return x() + 2 * planes * xn() * (1 + which); }
  __host__ __device__ int64_t am() const { return xt(2); }
  __host__ __device__ int64_t bm() const { return am() + 2 * planes * an(); }
  __host__ __device__ int64_t bytes() const { return bm() + 2 * planes * an(); }
};

__device__ __forceinline__ void split(float v, _Float16 &hi, _Float16 &lo) {
  hi = (_Float16)v;
  lo = (_Float16)(v - (float)hi);
}

template <class T> __global__ __launch_bounds__(NT) void k_os_norm(Args a) {
  __shared__ double s_[NT / 64];
  const Mat m = a.m[blockIdx.y];
  const int64_t n = (int64_t)m.rows * m.cols;
  double s = 0.0;
  for (int64_t i = blockIdx.x * (int64_t)NT + threadIdx.x; i < n; i += (int64_t)NORM_PARTS * NT) {
    const double v = to_f32(((const T *)m.in)[i]);
    s = fma(v, v, s);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
  if ((threadIdx.x & 63) == 0) s_[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) ((double *)(a.ws + m.ws))[blockIdx.x] = ((s_[0] + s_[1]) + s_[2]) + s_[3];
}

// block -> (matrix, tile of it) for a phase with tiles(lay) tiles a matrix
template <class F> __device__ __forceinline__ int find(const Args &a, int &tile, F tiles) {
  int m = 0;
  for (; m < a.count - 1; ++m) {
    const int t = tiles(Lay(a.m[m].rows, a.m[m].cols, a.planes));
    if (tile < t) break;
    tile -= t;
  }
  return m;
}

// X0 and its transpose, scaled, split and zero padded: one 64 x 64 tile of X a workgroup
template <class T> __global__ __launch_bounds__(NT) void k_os_pack(Args a) {
  __shared__ float t_[TILE][TILE + 1];
  int tile = blockIdx.x;
  const int mi = find(a, tile, [](const Lay &y) { return (y.sp / TILE) * (y.lp / TILE); });
  const Mat m = a.m[mi];
  const Lay y(m.rows, m.cols, a.planes);
  char *ws = a.ws + m.ws;
  double sum = 0.0;
  for (int i = 0; i < NORM_PARTS; ++i) sum += ((const double *)ws)[i];
  const double norm = sqrt(sum) + a.eps;
  const double scale = norm < 1e300 ? (norm > 0.0 ? (double)SX / norm : 0.0) : NAN;  // (no finite norm: no result)
  const int i0 = tile / (y.lp / TILE) * TILE, j0 = tile % (y.lp / TILE) * TILE, tid = threadIdx.x;
  for (int e = tid; e < TILE * TILE; e += NT) {
    const int p = e / TILE, q = e % TILE;  // q runs along M's rows
    const int r = y.tall ? j0 + p : i0 + p, c = y.tall ? i0 + q : j0 + q;
    float v = 0.0f;
    if (r < m.rows && c < m.cols) v = (float)((double)to_f32(((const T *)m.in)[(int64_t)r * m.cols + c]) * scale);
    if (y.tall) t_[q][p] = v;
    else t_[p][q] = v;
  }
  __syncthreads();
  _Float16 *x = (_Float16 *)(ws + y.x()), *xt = (_Float16 *)(ws + y.xt(0));
  for (int e = tid; e < TILE * TILE; e += NT) {
    const int p = e / TILE, q = e % TILE;
    _Float16 hi, lo;
    split(t_[p][q], hi, lo);
    x[(int64_t)(i0 + p) * y.lp + j0 + q] = hi;
    if (a.planes == 2) x[y.xn() + (int64_t)(i0 + p) * y.lp + j0 + q] = lo;
    split(t_[q][p], hi, lo);
    xt[(int64_t)(j0 + p) * y.sp + i0 + q] = hi;
    if (a.planes == 2) xt[y.xn() + (int64_t)(j0 + p) * y.sp + i0 + q] = lo;
  }
}

enum { GRAM, POLY, UPDATE, LAST };

template <int PHASE> __host__ __device__ __forceinline__ int tiles_of(const Lay &y) {
  const int s = y.sp / TILE, l = y.lp / TILE;
  return PHASE == GRAM || PHASE == POLY ? s * (s + 1) / 2 : s * l;
}

template <int PHASE, int P, class T> __global__ __launch_bounds__(NT) void k_os_gemm(Args a) {
  __shared__ __attribute__((aligned(16))) _Float16 sp_[P][TILE][PITCH], sq_[P][TILE][PITCH];
  int tile = blockIdx.x;
  const int mi = find(a, tile, [](const Lay &y) { return tiles_of<PHASE>(y); });
  const Mat m = a.m[mi];
  const Lay y(m.rows, m.cols, P);
  char *ws = a.ws + m.ws;
  int ti, tj;
  if (PHASE == GRAM || PHASE == POLY) {  // row ti holds the tiles tj >= ti
    ti = 0;
    for (int n = y.sp / TILE; tile >= n - ti; ++ti) tile -= n - ti;
    tj = ti + tile;
  } else {
    ti = tile % (y.sp / TILE);
    tj = tile / (y.sp / TILE);
  }
  const int i0 = ti * TILE, j0 = tj * TILE;
  const _Float16 *p, *q;
  int64_t pn, qn;
  int k_n;
  if (PHASE == GRAM) { p = q = (const _Float16 *)(ws + y.x()); pn = qn = y.xn(); k_n = y.lp; }
  else if (PHASE == POLY) { p = q = (const _Float16 *)(ws + y.am()); pn = qn = y.an(); k_n = y.sp; }
  else { p = (const _Float16 *)(ws + y.bm()); pn = y.an(); q = (const _Float16 *)(ws + y.xt(a.cur)); qn = y.xn(); k_n = y.sp; }
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wi = (wave >> 1) * 32, wj = (wave & 1) * 32;
  const int lr = tid >> 2, lk = (tid & 3) * 8;  // what this thread stages: 8 k of one row
  f32x16 acc = {};
  for (int k0 = 0; k0 < k_n; k0 += KS) {
    half8 vp[P], vq[P];
#pragma unroll
    for (int h = 0; h < P; ++h) {
      vp[h] = *(const half8 *)(p + h * pn + (int64_t)(i0 + lr) * k_n + k0 + lk);
      vq[h] = *(const half8 *)(q + h * qn + (int64_t)(j0 + lr) * k_n + k0 + lk);
    }
    __syncthreads();
#pragma unroll
    for (int h = 0; h < P; ++h) {
      *(half8 *)&sp_[h][lr][lk] = vp[h];
      *(half8 *)&sq_[h][lr][lk] = vq[h];
    }
    __syncthreads();
#pragma unroll
    for (int kk = 0; kk < KS; kk += 16) {
      half8 fp[P], fq[P];
#pragma unroll
      for (int h = 0; h < P; ++h) {
        fp[h] = *(const half8 *)&sp_[h][wi + (lane & 31)][kk + (lane >> 5) * 8];
        fq[h] = *(const half8 *)&sq_[h][wj + (lane & 31)][kk + (lane >> 5) * 8];
      }
      if (P == 2) {
        acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(fp[P - 1], fq[0], acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(fp[0], fq[P - 1], acc, 0, 0, 0);
      }
      acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(fp[0], fq[0], acc, 0, 0, 0);
    }
  }
  // lane: column j of the tile, rows in groups of four
  const int j = j0 + wj + (lane & 31);
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const int i = i0 + wi + (e >> 2) * 8 + (lane >> 5) * 4 + (e & 3);
    if (PHASE == GRAM || PHASE == POLY) {
      float v;
      if (PHASE == GRAM) v = acc[e] * (SA / (SX * SX));
      else {
        const int64_t at = (int64_t)i * y.sp + j;
        float av = (float)p[at];
        if (P == 2) av += (float)p[pn + at];
        v = fmaf(a.c / SA, acc[e], a.b * av);
      }
      _Float16 *o = (_Float16 *)(ws + (PHASE == GRAM ? y.am() : y.bm()));
      _Float16 hi, lo;
      split(v, hi, lo);
      o[(int64_t)i * y.sp + j] = hi;
      if (P == 2) o[y.an() + (int64_t)i * y.sp + j] = lo;
      if (ti != tj) {
        o[(int64_t)j * y.sp + i] = hi;
        if (P == 2) o[y.an() + (int64_t)j * y.sp + i] = lo;
      }
    } else {
      _Float16 *x = (_Float16 *)(ws + y.x());
      const int64_t at = (int64_t)i * y.lp + j;
      float xv = (float)x[at];
      if (P == 2) xv += (float)x[y.xn() + at];
      const float v = fmaf(a.a, xv, acc[e] * (1.0f / SA));
      if (PHASE == LAST) {
        if (i < y.s && j < y.l) from_f32(v * (1.0f / SX), ((T *)m.out)[y.tall ? (int64_t)j * m.cols + i : (int64_t)i * m.cols + j]);
      } else {
        _Float16 *xt = (_Float16 *)(ws + y.xt(a.cur ^ 1));
        _Float16 hi, lo;
        split(v, hi, lo);
        x[at] = hi;
        xt[(int64_t)j * y.sp + i] = hi;
        if (P == 2) { x[y.xn() + at] = lo; xt[y.xn() + (int64_t)j * y.sp + i] = lo; }
      }
    }
  }
}

static int64_t round_up(int64_t v) { return (v + 255) / 256 * 256; }

static int check(const char *&msg, int32_t dtype, int32_t count, const int32_t *rows, const int32_t *cols) {
  if (dtype != AZ_NN_F32 && dtype != AZ_NN_BF16 && dtype != AZ_NN_F16) { msg = "orthogonalize: unknown dtype"; return AZ_EINVAL; }
  if (count < 0 || (count > 0 && (!rows || !cols))) { msg = "orthogonalize: count >= 0, rows and cols given"; return AZ_EINVAL; }
  for (int i = 0; i < count; ++i)
    if (rows[i] < 0 || cols[i] < 0 || rows[i] > 65536 || cols[i] > 65536) { msg = "orthogonalize: sides of 0 .. 65,536"; return AZ_EINVAL; }
  return AZ_OK;
}

// Singular values stay in [0, top]: top of step k + 1 is the largest |a s + b s^3 + c s^5| over [0, top of step k].  The stored X, A and
// B are f16, so coefficients that let them grow without bound are refused.
static bool bounded(int steps, double a, double b, double c) {
  if (!std::isfinite(a) || !std::isfinite(b) || !std::isfinite(c)) return false;
  double top = 1.0;
  for (int k = 0; k < steps; ++k) {
    double next = 0.0, poly = 0.0;
    for (int i = 0; i <= 4096; ++i) {
      const double s = top * i / 4096.0, s2 = s * s;
      next = std::fmax(next, std::fabs(s * (a + s2 * (b + c * s2))));
      poly = std::fmax(poly, std::fabs(s2 * (b + c * s2)));
    }
    if (!(poly < 100.0) || !(next < 7.5)) return false;
    top = next * 1.001;
  }
  return true;
}

template <class T, int P> static int run(const Args &base, int steps, hipStream_t s) {
  Args a = base;
  int t[4] = {0, 0, 0, 0}, pack = 0;
  for (int i = 0; i < a.count; ++i) {
    const Lay y(a.m[i].rows, a.m[i].cols, P);
    t[GRAM] += tiles_of<GRAM>(y);
    t[UPDATE] += tiles_of<UPDATE>(y);
    pack += (y.sp / TILE) * (y.lp / TILE);
  }
  hipLaunchKernelGGL((k_os_norm<T>), dim3(NORM_PARTS, a.count), dim3(NT), 0, s, a);
  hipLaunchKernelGGL((k_os_pack<T>), dim3(pack), dim3(NT), 0, s, a);
  for (int k = 0; k < steps; ++k) {
    a.cur = k & 1;
    hipLaunchKernelGGL((k_os_gemm<GRAM, P, T>), dim3(t[GRAM]), dim3(NT), 0, s, a);
    hipLaunchKernelGGL((k_os_gemm<POLY, P, T>), dim3(t[GRAM]), dim3(NT), 0, s, a);
    if (k + 1 < steps) hipLaunchKernelGGL((k_os_gemm<UPDATE, P, T>), dim3(t[UPDATE]), dim3(NT), 0, s, a);
    else hipLaunchKernelGGL((k_os_gemm<LAST, P, T>), dim3(t[UPDATE]), dim3(NT), 0, s, a);
  }
  return launched("k_os");
}

}  // namespace azortho

extern "C" {

int64_t az_orthogonalize_workspace(int32_t dtype, int32_t count, const int32_t *rows, const int32_t *cols) {
  using namespace azortho;
  const char *msg = "";
  if (check(msg, dtype, count, rows, cols) != AZ_OK) { fail(AZ_EINVAL, msg); return -1; }
  int64_t total = 0;
  for (int i = 0; i < count; ++i)
    if (rows[i] > 0 && cols[i] > 0) total += round_up(Lay(rows[i], cols[i], dtype == AZ_NN_BF16 ? 1 : 2).bytes());
  return total;
}

int az_orthogonalize(int32_t dtype, int32_t count, const void *const *in, void *const *out, const int32_t *rows, const int32_t *cols,
                     int32_t steps, double a, double b, double c, double eps, void *workspace_dev, int64_t workspace_bytes, void *stream) {
  using namespace azortho;
  const char *msg = "";
  if (check(msg, dtype, count, rows, cols) != AZ_OK) return fail(AZ_EINVAL, msg);
  if (steps < 1 || steps > 64) return fail(AZ_EINVAL, "orthogonalize: 1 .. 64 steps");
  if (!(eps >= 0.0 && eps < 1e300)) return fail(AZ_EINVAL, "orthogonalize: eps >= 0");
  if (!bounded(steps, a, b, c)) return fail(AZ_EINVAL, "orthogonalize: these coefficients let singular values grow beyond 7.5 (or the polynomial beyond 100)");
  const int es = dtype == AZ_NN_F32 ? 4 : 2, planes = dtype == AZ_NN_BF16 ? 1 : 2;
  if (count > 0 && (!in || !out)) return fail(AZ_EINVAL, "orthogonalize: null argument");
  int live = 0;
  for (int i = 0; i < count; ++i) {
    if (rows[i] == 0 || cols[i] == 0) continue;
    ++live;
    if (!in[i] || !out[i] || misaligned(in[i], es) || misaligned(out[i], es)) return fail(AZ_EINVAL, "orthogonalize: null or misaligned matrix");
  }
  if (live == 0) return AZ_OK;
  if (!workspace_dev || misaligned(workspace_dev, 256) || workspace_bytes < az_orthogonalize_workspace(dtype, count, rows, cols))
    return fail(AZ_EINVAL, "orthogonalize: workspace below az_orthogonalize_workspace() or not aligned to 256 bytes");
  hipStream_t s = (hipStream_t)stream;
  DeviceGuard guard(s);
  if (!guard.ok) return fail(AZ_EHIP, "orthogonalize: cannot select the stream's device");
  Args g{};
  g.ws = (char *)workspace_dev;
  g.planes = planes;
  g.a = (float)a; g.b = (float)b; g.c = (float)c; g.eps = eps;
  uint64_t off = 0;
  for (int i = 0; i < count; ++i) {
    if (rows[i] == 0 || cols[i] == 0) continue;
    g.m[g.count++] = Mat{in[i], out[i], off, rows[i], cols[i]};
    off += (uint64_t)round_up(Lay(rows[i], cols[i], planes).bytes());
    --live;
    if (g.count == MAX_M || live == 0) {
      const int rc = dtype == AZ_NN_F32 ? run<float, 2>(g, steps, s) : dtype == AZ_NN_BF16 ? run<bf16_t, 1>(g, steps, s) : run<f16_t, 2>(g, steps, s);
      if (rc != AZ_OK) return rc;
      g.count = 0;
    }
  }
  return AZ_OK;
}

}  // extern "C"
