// az_ortho.hip -- orthogonalising updates by Newton-Schulz products, a whole network's matrices per call (gfx950).
//
//   X0 = M / (|M|_F + eps), transposed if M has more rows than columns (S = short side, L = long side);
//   per step:  A = X X^T,   B = b A + c A^2,   X <- a X + B X
//
// All three are products of the form C[i][j] = sum_k P[i][k] Q[j][k] with k consecutive in both operands: A from X with itself, A^2
// from the symmetric A with itself, B X from B and the transpose of X, which every step writes beside X.  Of the symmetric results
// only the tiles that touch the upper triangle are computed; the lower one is its mirror image.
//
// Arithmetic: f16 matrix instructions with f32 sums.  An operand is a pair of f16, hi = f16(v) and lo = f16(v - hi), and a product is
// hi hi + hi lo + lo hi: 22 bits of each factor, three matrix instructions, several times the rate of the f32 ones.  For bf16 matrices
// with a short side beyond 64 hi alone holds more (11 bits) than the result will (8; what that costs stands at planes_of).  Stored values
// are scaled by powers of two, as large as the host's bound on the singular values allows (az_orthogonalize: entries stay below 2^15),
// which keeps lo clear of f16's smallest steps.  Buffers are zero padded to whole tiles and the padding stays zero: no product has a
// border case.
//
// A row of an operand is a run of 128-byte units: 64 k of hi, or hi and lo of 32 k.  A stage of a product is one unit of every row of
// the two panels, moved straight from memory to LDS (16 bytes a lane) while the stage before it is multiplied.  Unit r's 16-byte
// pieces lie at piece ^ (r & 7), so that the 8 rows a quarter wave reads at once fall on different banks.
//
// Measured (a large f16 product by the library reaches 1,116 TFLOP/s on this card, a bf16 one 1,169):
//   4096 x 4096 bf16:                  1.74 ms; X 154 .. 166 us (137 GFLOP: 0.87 PFLOP/s), A and B 92 and 96 us (half of that: 0.73)
//   2501 x 1203 f32:                   451 us; X 42 us (22.2 GFLOP executed in three products of halves: 0.53 PFLOP/s): 1.5 tiles a slot
//   the deep 128-channel net's 23 f32: 183 us in 22 launches: 13 us for X (4.7 GFLOP executed), 9 + 5 for A, 6 for B: launches, and 752 tiles of
//                                      4 stages each, whose start and end weigh as much as their products
//   1536 x 1536 bf16 / f32:            260 / 489 us; 2000 x 4096 bf16 / f32: 615 / 1,348 us
//   64 x 576 f32 or bf16:              54 us in one launch, 11 a step: latencies of one workgroup (below)
#include "az_ops.hip.h"

#include <cmath>

namespace azortho {

using namespace azops;

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int NT = 256, MAX_M = 64, NORM_PARTS = 256, UNIT = 128;

struct Mat {
  const void *in;
  void *out;
  uint64_t ws;  // byte offset of this matrix's buffers
  int32_t rows, cols;
};
enum { GRAM, POLY, UPDATE, LAST };  // (POLY has GRAM's tiles, LAST has UPDATE's)
enum { WHOLE, SPLIT, JOIN };  // a tile's product at once; that, or for tiles from `whole` on a share of its k range; the shares' sum and what follows a product
struct Table {  // what the first launch carries and leaves at the start of the workspace for the others
  Mat m[MAX_M];
  uint32_t start[6][MAX_M];  // first tile of each matrix: of A and B, of X, of PACK; share of a cut tile; cut tile; tile done at once
  int32_t shares[MAX_M];     // of a cut tile's k range
  int32_t count;
};
struct Args {
  char *ws;  // Table, then the matrices' buffers
  float a, b, c;
  float sx, sa, sb;  // powers of two: the stored X, A and B are sx, sa and sb times theirs
  double eps;
  int32_t count, cur;
  int32_t n[6];     // tiles in all, as in Table::start
  uint64_t part;    // byte offset of the partial tiles
};

// one matrix's buffers: norm parts (f64), X, two transposes of X, A, B.  SP, LP: the sides padded.
struct Lay {
  int s, l, sp, lp, planes;
  bool tall;
  __host__ __device__ Lay(int rows, int cols, int planes_, int pad) {
    tall = rows > cols;
    s = tall ? cols : rows;
    l = tall ? rows : cols;
    sp = (s + pad - 1) / pad * pad;
    lp = (l + pad - 1) / pad * pad;
    planes = planes_;
  }
  __host__ __device__ int64_t xb() const { return (int64_t)sp * lp * 2 * planes; }  // bytes of X
  __host__ __device__ int64_t ab() const { return (int64_t)sp * sp * 2 * planes; }
  __host__ __device__ int64_t x() const { return NORM_PARTS * 8; }
  __host__ __device__ int64_t xt(int which) const { return x() + xb() * (1 + which); }
  __host__ __device__ int64_t am() const { return xt(2); }
  __host__ __device__ int64_t bm() const { return am() + ab(); }
  __host__ __device__ int64_t bytes() const { return bm() + ab(); }
};

// element (row, k) of an operand with K columns: hi, and 32 elements behind it lo
template <int P> __device__ __forceinline__ int64_t at(int64_t row, int k, int K) {
  return P == 1 ? row * K + k : row * 2 * K + (k >> 5) * 64 + (k & 31);
}
// eight consecutive k (a multiple of eight): 16 bytes of each plane
template <int P> __device__ __forceinline__ void put8(_Float16 *o, const float *v) {
  half8 hi, lo;
#pragma unroll
  for (int e = 0; e < 8; ++e) { hi[e] = (_Float16)v[e]; lo[e] = (_Float16)(v[e] - (float)hi[e]); }
  *(half8 *)o = hi;
  if (P == 2) *(half8 *)(o + 32) = lo;
}
template <int P> __device__ __forceinline__ void get8(const _Float16 *o, float *v) {
  const half8 hi = *(const half8 *)o;
  half8 lo = {};
  if (P == 2) lo = *(const half8 *)(o + 32);
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = (float)hi[e] + (float)lo[e];
}

// the workgroups that sum one matrix's squares, 16 Ki elements each: by the matrix alone (the order of a sum is part of its result)
__host__ __device__ __forceinline__ int parts_of(int rows, int cols) {
  const int64_t want = ((int64_t)rows * cols + 16383) / 16384;
  return (int)(want < NORM_PARTS ? want : NORM_PARTS);
}

// a row of workgroups a matrix, as long as the largest one's
template <class T> __global__ __launch_bounds__(NT) void k_os_norm(Table t, char *ws) {
  __shared__ double s_[NT / 64];
  const int tid = threadIdx.x;
  if (blockIdx.x == 0 && blockIdx.y == 0)
    for (int i = tid; i < (int)(sizeof(Table) / 4); i += NT) ((uint32_t *)ws)[i] = ((const uint32_t *)&t)[i];
  const Mat m = t.m[blockIdx.y];
  const int parts = parts_of(m.rows, m.cols);
  if ((int)blockIdx.x >= parts) return;
  const int64_t n = (int64_t)m.rows * m.cols;
  constexpr int V = 16 / sizeof(T);
  const int64_t nv = n / V;
  double s = 0.0;
  const T *in = (const T *)m.in;
#pragma unroll 4
  for (int64_t i = blockIdx.x * (int64_t)NT + tid; i < nv; i += (int64_t)parts * NT) {
    u32x4 w;
    __builtin_memcpy(&w, in + i * V, 16);  // (aligned to its elements only)
#pragma unroll
    for (int j = 0; j < V; ++j) { const double v = Word<T>::get(w[j / Word<T>::N], j % Word<T>::N); s = fma(v, v, s); }
  }
  for (int64_t i = nv * V + blockIdx.x * (int64_t)NT + tid; i < n; i += (int64_t)parts * NT) {
    const double v = to_f32(in[i]);
    s = fma(v, v, s);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
  if ((tid & 63) == 0) s_[tid >> 6] = s;
  __syncthreads();
  if (tid == 0) ((double *)(ws + m.ws))[blockIdx.x] = ((s_[0] + s_[1]) + s_[2]) + s_[3];
}

// Workgroups go round the 8 XCDs in turn; block b takes item (b % 8) * ceil(n / 8) + b / 8 of n, so that an XCD (and its L2) gets a
// run of neighbouring tiles, and much the same matrices in every phase.  -> -1: none (the grid is rounded up to whole turns)
__device__ __forceinline__ int item_of(int n, int block) {
  const int per = (n + 7) / 8, t = (block & 7) * per + (block >> 3);
  return (block >> 3) < per && t < n ? t : -1;
}
__host__ __device__ static inline unsigned grid_of(uint32_t n) { return (n + 7) / 8 * 8; }

// tile -> (matrix, tile of it): the lanes look at one matrix's first tile each
__device__ __forceinline__ int find(const Args &a, int kind, int &tile) {
  const uint32_t *start = ((const Table *)a.ws)->start[kind];
  const int lane = threadIdx.x & 63;
  const uint32_t mine = lane < a.count ? start[lane] : 0xFFFFFFFFu;
  const int m = __popcll(__ballot(mine <= (uint32_t)tile)) - 1;
  tile -= (int)__shfl(mine, m);
  tile = __builtin_amdgcn_readfirstlane(tile);
  return __builtin_amdgcn_readfirstlane(m);
}

// X0 and its transpose, scaled, split and zero padded: one 64 x 64 tile of X a workgroup
template <class T, int P, int PADT> __global__ __launch_bounds__(NT) void k_os_pack(Args a) {
  __shared__ float t_[64][65];
  __shared__ double s_[NT / 64];
  int tile = item_of(a.n[2], blockIdx.x);
  if (tile < 0) return;
  const int tid = threadIdx.x, mi = find(a, 2, tile);
  const Mat m = ((const Table *)a.ws)->m[mi];
  const Lay y(m.rows, m.cols, P, PADT);
  char *ws = a.ws + m.ws;
  double sum = tid < parts_of(m.rows, m.cols) ? ((const double *)ws)[tid] : 0.0;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
  if ((tid & 63) == 0) s_[tid >> 6] = sum;
  __syncthreads();
  sum = ((s_[0] + s_[1]) + s_[2]) + s_[3];
  const double norm = sqrt(sum) + a.eps;
  const double scale = norm < 1e300 ? (norm > 0.0 ? (double)a.sx / norm : 0.0) : NAN;  // (no finite norm: no result)
  const int i0 = tile / (y.lp / 64) * 64, j0 = tile % (y.lp / 64) * 64;
  for (int e = tid; e < 64 * 64; e += NT) {
    const int p = e / 64, q = e % 64;  // q runs along M's rows
    const int r = y.tall ? j0 + p : i0 + p, c = y.tall ? i0 + q : j0 + q;
    float v = 0.0f;
    if (r < m.rows && c < m.cols) v = (float)((double)to_f32(((const T *)m.in)[(int64_t)r * m.cols + c]) * scale);
    if (y.tall) t_[q][p] = v;
    else t_[p][q] = v;
  }
  __syncthreads();
  _Float16 *x = (_Float16 *)(ws + y.x()), *xt = (_Float16 *)(ws + y.xt(0));
  for (int e = tid; e < 64 * 8; e += NT) {
    const int p = e / 8, q = e % 8 * 8;
    float v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = t_[p][q + k];
    put8<P>(x + at<P>(i0 + p, j0 + q, y.lp), v);
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = t_[q + k][p];
    put8<P>(xt + at<P>(j0 + p, i0 + q, y.sp), v);
  }
}

// 1 KiB from memory to LDS: 16 bytes a lane, at lds + 16 lane
__device__ __forceinline__ void to_lds(const char *base, uint32_t lane_off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" : : "s"(lds), "v"(lane_off), "s"(base) : "memory", "m0");
}
// all but the newest N of this wave's moves have landed and its LDS reads are done, then the workgroup goes on
template <int N> __device__ __forceinline__ void stage_barrier() { asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" : : "n"(N) : "memory"); }

// the wave's LDS writes are seen by its other lanes
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// row ti of the upper triangle of an n x n grid of tiles holds tj = ti .. n - 1
__device__ __forceinline__ void upper(int tile, int n, int &ti, int &tj) {
  // the row starts at ti n - ti (ti - 1) / 2
  ti = (int)(((float)(2 * n + 1) - sqrtf((float)(2 * n + 1) * (float)(2 * n + 1) - 8.0f * (float)tile)) * 0.5f);
  ti = ti < 0 ? 0 : ti > n - 1 ? n - 1 : ti;
  while (ti > 0 && ti * n - ti * (ti - 1) / 2 > tile) --ti;
  while (ti < n - 1 && (ti + 1) * n - (ti + 1) * ti / 2 <= tile) ++ti;
  tj = ti + tile - (ti * n - ti * (ti - 1) / 2);
}

// Tile of an ni x nj grid walked in bands of 8 rows, column by column: the 64 tiles that an XCD works on at a time read 16 panels of their
// operands, not 34 (4096 x 4096 bf16: 155 us against 162 in columns of 32; bands of 4 and 16 are no better)
__device__ __forceinline__ void square(int tile, int ni, int nj, int &ti, int &tj) {
  const int band = tile / (8 * nj), in = tile - band * 8 * nj, rows = min(8, ni - band * 8);
  tj = in / rows;
  ti = band * 8 + in - tj * rows;
}

template <int PHASE> __host__ __device__ __forceinline__ int tiles_of(const Lay &y, int t) {
  const int s = y.sp / t, l = y.lp / t;
  return PHASE == GRAM || PHASE == POLY ? s * (s + 1) / 2 : s * l;
}

// Which of A's tiles are cut along k, by the matrix alone (its result must not depend on the others in the call): those from `whole` on, in
// `shares` each.
//   tiles of 64: at most 96 of them leave CUs idle, and with 32 stages or more a share of 8 stages or more is worth the second pass; A only.
//   (Up to 256 tiles in two or more shares: 900 x 8000 f32 850 -> 701 us, but 2501 x 1203 465 -> 472, four of 900 x 2000 745 -> 812.)
//   tiles of 128: two workgroups a CU hold 512 at a time (one plane), one 256 (two planes); what little is left over after whole turns would
//   take a turn of its own.  B = A A as well (its k range is the short side, 28 stages or more).  4096 x 4096 bf16, 528 tiles: 112 us at once,
//   97 with the last 16 in four shares each (102 in two, 105 in sixteen: those wait for the join).
struct Split { int whole, shares; };
__host__ __device__ __forceinline__ Split split_of(const Lay &y, int tile) {
  const int tiles = tiles_of<GRAM>(y, tile);
  if (tile == 64) {
    const int stages = y.lp * 2 * y.planes / UNIT;
    if (tiles > 96 || stages < 32) return Split{tiles, 1};
    const int s = 512 / tiles < stages / 8 ? 512 / tiles : stages / 8;
    return Split{s > 1 ? 0 : tiles, s < 8 ? s : 8};
  }
  const int turn = y.planes == 1 ? 512 : 256, left = tiles % turn;
  if (tiles < turn || left == 0 || left > turn / 4) return Split{tiles, 1};
  return Split{tiles - left, 4};
}

// One T x T tile, four waves, (T / 2) x (T / 2) each in blocks of 32 x 32.  T = 64, and T = 128 with two planes, which leaves a CU one
// workgroup: four stages in LDS, the moves of three under way while one is multiplied.  T = 128 with one plane: two stages, and two
// workgroups a CU cover for each other.
// Tiles of A (and of B) may be cut along k (split_of): every share leaves its sums as they lie in its registers, and JOIN adds the shares in
// order and goes on as WHOLE does.
template <int PHASE, int P, int T, class E, int MODE> __global__ __launch_bounds__(NT) void k_os_gemm(Args a) {
  constexpr bool SYM = PHASE == GRAM || PHASE == POLY;
  constexpr int B = T / 64, W = T / 2, STAGE = 2 * T * UNIT, BUFS = T == 64 || P == 2 ? 4 : 2, MOVES = 2 * T / 8 / 4;
  __shared__ __attribute__((aligned(1024))) char lds[BUFS * STAGE];
  // SPLIT: the tiles done at once, then the shares of the others (shorter, they fill what the last of those leave idle)
  const int ahead = MODE == SPLIT ? (int)grid_of(a.n[5]) : 0;
  const bool part = MODE == SPLIT && (int)blockIdx.x >= ahead;
  const int kind = MODE == SPLIT ? (part ? 3 : 5) : MODE == JOIN ? 4 : SYM ? 0 : 1;
  int tile = item_of(a.n[kind], part ? blockIdx.x - ahead : blockIdx.x);
  if (tile < 0) return;
  const int mi = find(a, kind, tile);
  const int shares = MODE == JOIN || part ? ((const Table *)a.ws)->shares[mi] : 1, share = part ? tile % shares : 0;
  const int64_t first = MODE == WHOLE ? 0 : (int64_t)((const Table *)a.ws)->start[3][mi] + (int64_t)tile * (part ? 1 : shares);  // its sums
  const Mat m = ((const Table *)a.ws)->m[mi];
  const Lay y(m.rows, m.cols, P, T);
  char *ws = a.ws + m.ws;
  if (MODE == JOIN || part) tile = split_of(y, T).whole + tile / (part ? shares : 1);
  int ti, tj;
  if (SYM) upper(tile, y.sp / T, ti, tj);
  else square(tile, y.sp / T, y.lp / T, ti, tj);
  const int i0 = ti * T, j0 = tj * T, K = PHASE == GRAM ? y.lp : y.sp, pitch = K * 2 * P, stages = pitch / UNIT;
  const char *p, *q;
  if (PHASE == GRAM) p = q = ws + y.x();
  else if (PHASE == POLY) p = q = ws + y.am();
  else { p = ws + y.bm(); q = ws + y.xt(a.cur); }
  p += (int64_t)i0 * pitch;
  q += (int64_t)j0 * pitch;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), wi = (wave >> 1) * (T / 2), wj = (wave & 1) * (T / 2);
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)lds;
  const uint32_t lane_off = (uint32_t)((lane >> 3) * pitch + (((lane & 7) ^ (lane >> 3)) << 4));
  auto issue = [&](int stage) {
    const uint32_t dst = lds0 + (stage & (BUFS - 1)) * STAGE;
#pragma unroll
    for (int e = 0; e < MOVES; ++e) {
      const int g = e * 4 + wave;  // eight rows of P's panel, or of Q's
      const char *src = (g < T / 8 ? p + (int64_t)g * 8 * pitch : q + (int64_t)(g - T / 8) * 8 * pitch) + (int64_t)stage * UNIT;
      to_lds(src, lane_off, dst + g * 1024);
    }
  };
  f32x16 acc[B][B] = {}, low[P == 2 ? B : 1][P == 2 ? B : 1] = {};  // hi hi; hi lo + lo hi, joined at the end: a third of the roundings
  const int rp = (wi + (lane & 31)) * UNIT, rq = (T + wj + (lane & 31)) * UNIT, sw = lane & 7, hf = lane >> 5;
  if constexpr (MODE != JOIN) {
  const int s0 = part ? (int)((int64_t)stages * share / shares) : 0, s1 = part ? (int)((int64_t)stages * (share + 1) / shares) : stages;
#pragma unroll
  for (int s = 0; s < BUFS - 1; ++s)
    if (s0 + s < s1) issue(s0 + s);
  for (int s = s0; s < s1; ++s) {
    // stage s is here (younger ones may be under way), and stage s - 1 has been read by every wave: its buffer takes stage s + BUFS - 1
    if (s + BUFS - 2 < s1) stage_barrier<(BUFS - 2) * MOVES>();
    else stage_barrier<0>();
    if (s + BUFS - 1 < s1) issue(s + BUFS - 1);
    const char *base = lds + (s & (BUFS - 1)) * STAGE;
#pragma unroll
    for (int kk = 0; kk < 4 / P; ++kk) {
      half8 fp[B][P], fq[B][P];
#pragma unroll
      for (int h = 0; h < P; ++h) {
        const int piece = ((h * 4 + kk * 2 + hf) ^ sw) << 4;
#pragma unroll
        for (int x = 0; x < B; ++x) {
          fp[x][h] = *(const half8 *)(base + rp + x * 32 * UNIT + piece);
          fq[x][h] = *(const half8 *)(base + rq + x * 32 * UNIT + piece);
        }
      }
#pragma unroll
      for (int x = 0; x < B; ++x)
#pragma unroll
        for (int z = 0; z < B; ++z) {
          if (P == 2) {
            low[x][z] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fp[x][P - 1], fq[z][0], low[x][z], 0, 0, 0);
            low[x][z] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fp[x][0], fq[z][P - 1], low[x][z], 0, 0, 0);
          }
          acc[x][z] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fp[x][0], fq[z][0], acc[x][z], 0, 0, 0);
        }
    }
  }
  stage_barrier<0>();
  }
  if (MODE == JOIN || part) {
    // [tile][share][block][element][thread] f32
    constexpr int64_t STEP = (int64_t)B * B * 16 * NT;
    float *sums = (float *)(a.ws + a.part) + first * STEP + tid;
    for (int k = 0; k < (MODE == JOIN ? shares : 1); ++k) {
#pragma unroll
      for (int x = 0; x < B; ++x)
#pragma unroll
        for (int z = 0; z < B; ++z)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            float *q_ = sums + ((x * B + z) * 16 + e) * NT;
            if (MODE == JOIN) acc[x][z][e] += *q_;
            else *q_ = P == 2 ? acc[x][z][e] + low[x][z][e] : acc[x][z][e];
          }
      sums += STEP;
    }
    if (MODE != JOIN) return;
  }
  // The results go through LDS, 32 rows of a wave's share at a time (a wave uses its own strip only), so that memory sees whole units:
  // first row by row, where the term a X or b A is added, then column by column for the mirror image or the transpose.
  constexpr int SP_ = W + 1;
  float *strip = (float *)lds + wave * 32 * SP_;
  static_assert(4 * 32 * SP_ * 4 <= BUFS * STAGE, "the strips fit the stages' memory");
#pragma unroll
  for (int x = 0; x < B; ++x) {
    // a lane holds column lane % 32 of a block, rows in groups of four
#pragma unroll
    for (int z = 0; z < B; ++z)
#pragma unroll
      for (int e = 0; e < 16; ++e) strip[((e >> 2) * 8 + hf * 4 + (e & 3)) * SP_ + z * 32 + (lane & 31)] = P == 2 ? acc[x][z][e] + low[x][z][e] : acc[x][z][e];
    wave_sync();
    const int r0 = i0 + wi + x * 32, c0 = j0 + wj;
    for (int e = lane; e < 32 * W / 8; e += 64) {
      const int r = e / (W / 8), c = e % (W / 8) * 8;
      float v[8], old[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = strip[r * SP_ + c + k];
      if (PHASE == GRAM) {
        const float f = a.sa / (a.sx * a.sx);
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] *= f;
        put8<P>((_Float16 *)(ws + y.am()) + at<P>(r0 + r, c0 + c, y.sp), v);
      } else if (PHASE == POLY) {
        get8<P>((const _Float16 *)(ws + y.am()) + at<P>(r0 + r, c0 + c, y.sp), old);
        const float f = a.c * (a.sb / (a.sa * a.sa)), g = a.b * (a.sb / a.sa);
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = fmaf(f, v[k], g * old[k]);
        put8<P>((_Float16 *)(ws + y.bm()) + at<P>(r0 + r, c0 + c, y.sp), v);
      } else {
        _Float16 *o = (_Float16 *)(ws + y.x()) + at<P>(r0 + r, c0 + c, y.lp);
        get8<P>(o, old);
        const float f = 1.0f / a.sb;
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = fmaf(a.a, old[k], v[k] * f);
        if (PHASE == UPDATE) put8<P>(o, v);
      }
      if (PHASE != GRAM || ti != tj) {
#pragma unroll
        for (int k = 0; k < 8; ++k) strip[r * SP_ + c + k] = v[k];
      }
    }
    wave_sync();
    if (PHASE == LAST) {  // rows and columns inside the matrix, in its own orientation
      const float f = 1.0f / a.sx;
      for (int e = lane; e < 32 * W; e += 64) {
        const int r = y.tall ? e % 32 : e / W, c = y.tall ? e / 32 : e % W, i = r0 + r, j = c0 + c;
        if (i < y.s && j < y.l) from_f32(strip[r * SP_ + c] * f, ((E *)m.out)[y.tall ? (int64_t)j * m.cols + i : (int64_t)i * m.cols + j]);
      }
    } else if (!SYM || ti != tj) {
      _Float16 *o = (_Float16 *)(ws + (PHASE == GRAM ? y.am() : PHASE == POLY ? y.bm() : y.xt(a.cur ^ 1)));
      for (int e = lane; e < W * 4; e += 64) {
        const int c = e / 4, r = e % 4 * 8;
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = strip[(r + k) * SP_ + c];
        put8<P>(o + at<P>(c0 + c, r0 + r, y.sp), v);
      }
    }
    wave_sync();
  }
}

// ---------------------------------------------------------------------------------------------------- one workgroup a matrix
// A short side of at most 64 and a long one of at most 768: X stays in registers for all steps (its f16 halves, in 32 x 32 blocks as the
// matrix instructions leave them: a lane holds a column's rows in groups of four), eight waves own every eighth column block.  Nothing but A
// and B passes through LDS, and one launch replaces 17: those matrices' steps are bound by launches and latencies.
//   B X: the block's own rows are the second factor as they lie; the first (rows of B) is read in the same order of k.
//   X X^T needs X with a lane holding a row: the block times the identity, which moves every f16 half unchanged.
// Partial sums of A go through LDS (four waves' at a time, always added in one order), waves 0 .. 2 take a tile of A and B each.
constexpr int SMALL_S = 64, SMALL_L = 768, SMALL_NT = 512, SMALL_NB = 3;

struct SmallTable {
  Mat m[MAX_M];
};

// piece q (four halves) of row r of a 64 x 64 f16 plane; the pieces of 16 rows fall on different banks
__device__ __forceinline__ int piece(int r, int q) { return r * 64 + ((q ^ (r & 15)) << 2); }

template <class E, int RB> __global__ __launch_bounds__(SMALL_NT) void k_os_small(SmallTable t, float ca, float cb, float cc, double eps, float sx, float sa, float sb, int steps) {
  constexpr int TILES = RB == 1 ? 1 : 3;
  __shared__ __attribute__((aligned(16))) char lds[4 * TILES * 16 * 64 * 4 + 64 * 64 * 4];
  float *part = (float *)lds;                                         // [slot 4][tile][element 16][lane]
  _Float16 *am = (_Float16 *)(lds + 4 * TILES * 16 * 64 * 4);         // A: planes of 64 x 64
  _Float16 *bm = (_Float16 *)lds;                                     // B: over the partial sums, which have been read by then
  static_assert(64 * 64 * 4 <= 4 * TILES * 16 * 64 * 4, "B fits the partial sums' memory");
  const Mat m = t.m[blockIdx.x];
  const bool tall = m.rows > m.cols;
  const int S = tall ? m.cols : m.rows, L = tall ? m.rows : m.cols;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), hf = lane >> 5, l32 = lane & 31;
  const int blocks = (L + 31) / 32, nb = wave < blocks ? (blocks - wave + 7) / 8 : 0;
  u32x4 x[SMALL_NB][RB][2][2];  // [block][32 rows][chunk of 16 rows][hi, lo], two f16 a word
  f32x16 raw[SMALL_NB][RB];
  double sum = 0.0;
#pragma unroll
  for (int b = 0; b < SMALL_NB; ++b)
#pragma unroll
    for (int r = 0; r < RB; ++r)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int j = (wave + 8 * b) * 32 + l32, i = r * 32 + (e >> 2) * 8 + hf * 4 + (e & 3);
        const int jc = min(j, L - 1), ic = min(i, S - 1);  // (every load at once, from inside the matrix)
        const float in = to_f32(((const E *)m.in)[(uint32_t)(tall ? jc * S + ic : ic * L + jc)]), v = j < L && i < S ? in : 0.0f;
        raw[b][r][e] = v;
        sum = fma((double)v, (double)v, sum);
      }
  {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
    double *s_ = (double *)lds;
    if (lane == 0) s_[wave] = sum;
    __syncthreads();
    sum = 0.0;
    for (int w = 0; w < 8; ++w) sum += s_[w];
    __syncthreads();
  }
  const double norm = sqrt(sum) + eps;
  const double scale = norm < 1e300 ? (norm > 0.0 ? (double)sx / norm : 0.0) : NAN;  // (no finite norm: no result)
  typedef _Float16 half2_ __attribute__((ext_vector_type(2)));
  auto keep = [&](u32x4 (&o)[2][2], int e, float v0, float v1) {  // elements e and e + 1
    const half2_ hi = {(_Float16)v0, (_Float16)v1};
    o[e >> 3][0][(e & 7) >> 1] = __builtin_bit_cast(uint32_t, hi);
    o[e >> 3][1][(e & 7) >> 1] = __builtin_bit_cast(uint32_t, half2_{(_Float16)(v0 - (float)hi[0]), (_Float16)(v1 - (float)hi[1])});
  };
  auto packed = [&](u32x4 (&o)[2][2]) {  // (whole words from here on, not an element a register)
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int h = 0; h < 2; ++h) asm volatile("" : "+v"(o[c][h]));
  };
#pragma unroll
  for (int b = 0; b < SMALL_NB; ++b)
#pragma unroll
    for (int r = 0; r < RB; ++r) {
#pragma unroll
      for (int e = 0; e < 16; e += 2) {
        const int j = (wave + 8 * b) * 32 + l32, i = r * 32 + (e >> 2) * 8 + hf * 4 + (e & 3);
        const bool in = b < nb && j < L;
        keep(x[b][r], e, in && i < S ? (float)((double)raw[b][r][e] * scale) : 0.0f, in && i + 1 < S ? (float)((double)raw[b][r][e + 1] * scale) : 0.0f);
      }
      packed(x[b][r]);
    }
  // the identity in the order of k that a block's rows have: place (hf, j) of chunk c is row 16 c + (j / 4) * 8 + hf * 4 + j % 4
  half8 one[2];
#pragma unroll
  for (int c = 0; c < 2; ++c)
#pragma unroll
    for (int j = 0; j < 8; ++j) one[c][j] = (_Float16)(16 * c + (j >> 2) * 8 + hf * 4 + (j & 3) == l32 ? 1.0f : 0.0f);
  // rows r * 32 .. of a symmetric 64 x 64 plane pair as the first factor, chunk c of its columns in that order of k
  auto rows_of = [&](const _Float16 *p, int r, int c, int h) {
    const _Float16 *q = p + h * 4096;
    const half4 u = *(const half4 *)(q + piece(r * 32 + l32, c * 4 + hf)), v = *(const half4 *)(q + piece(r * 32 + l32, c * 4 + 2 + hf));
    return half8{u[0], u[1], u[2], u[3], v[0], v[1], v[2], v[3]};
  };
  // a tile of a symmetric matrix into the planes: columns (four consecutive rows a lane), and off the diagonal its mirror image
  auto put_tile = [&](_Float16 *p, const float *v, int ti, int tj) {
#pragma unroll
    for (int e4 = 0; e4 < 4; ++e4) {
      half4 hi, lo;
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        hi[d] = (_Float16)v[e4 * 4 + d];
        lo[d] = (_Float16)(v[e4 * 4 + d] - (float)hi[d]);
      }
      const int j = tj * 32 + l32, i = ti * 32 + e4 * 8 + hf * 4;
      *(half4 *)(p + piece(j, i >> 2)) = hi;
      *(half4 *)(p + 4096 + piece(j, i >> 2)) = lo;
      if (ti != tj) {
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          p[piece(i + d, j >> 2) + (j & 3)] = hi[d];
          p[4096 + piece(i + d, j >> 2) + (j & 3)] = lo[d];
        }
      }
    }
  };
  for (int step = 0; step < steps; ++step) {
    // A's share of this wave's columns
    f32x16 acc[TILES] = {};
#pragma unroll
    for (int b = 0; b < SMALL_NB; ++b) {
      if (b >= nb) continue;
      half8 xt[RB][2][2];
#pragma unroll
      for (int r = 0; r < RB; ++r)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          f32x16 d = {};
          d = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8, x[b][r][0][h]), one[0], d, 0, 0, 0);
          d = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8, x[b][r][1][h]), one[1], d, 0, 0, 0);
#pragma unroll
          for (int c = 0; c < 2; ++c) {  // (the values are f16 already: no rounding)
            u32x4 w;
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(d[c * 8 + 2 * j], d[c * 8 + 2 * j + 1]));
            xt[r][c][h] = __builtin_bit_cast(half8, w);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
      for (int q = 0; q < TILES; ++q) {
        const int ti = q == 2 ? 1 : 0, tj = q == 0 ? 0 : 1;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          acc[q] = __builtin_amdgcn_mfma_f32_32x32x16_f16(xt[ti][c][1], xt[RB == 1 ? 0 : tj][c][0], acc[q], 0, 0, 0);
          acc[q] = __builtin_amdgcn_mfma_f32_32x32x16_f16(xt[ti][c][0], xt[RB == 1 ? 0 : tj][c][1], acc[q], 0, 0, 0);
          acc[q] = __builtin_amdgcn_mfma_f32_32x32x16_f16(xt[ti][c][0], xt[RB == 1 ? 0 : tj][c][0], acc[q], 0, 0, 0);
        }
      }
    }
    __syncthreads();  // (B of the step before has been read)
    auto slot = [&](int q, int e) { return part + (((wave & 3) * TILES + q) * 16 + e) * 64 + lane; };
    if (wave >= 4) {
#pragma unroll
      for (int q = 0; q < TILES; ++q)
#pragma unroll
        for (int e = 0; e < 16; ++e) *slot(q, e) = acc[q][e];
    }
    __syncthreads();
    if (wave < 4) {
#pragma unroll
      for (int q = 0; q < TILES; ++q)
#pragma unroll
        for (int e = 0; e < 16; ++e) *slot(q, e) += acc[q][e];
    }
    __syncthreads();
    const int ti = wave == 2 ? 1 : 0, tj = wave == 0 || RB == 1 ? 0 : 1;  // waves 0 .. TILES - 1: their tile
    float a[16];
    if (wave < TILES) {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        float v = 0.0f;
#pragma unroll
        for (int s = 0; s < 4; ++s) v += part[((s * TILES + wave) * 16 + e) * 64 + lane];
        a[e] = v * (sa / (sx * sx));
      }
      put_tile(am, a, ti, tj);
    }
    __syncthreads();
    if (wave < TILES) {
      f32x16 d = {};
#pragma unroll
      for (int c = 0; c < 2 * RB; ++c) {
        half8 p[2], q[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) { p[h] = rows_of(am, ti, c, h); q[h] = rows_of(am, tj, c, h); }
        d = __builtin_amdgcn_mfma_f32_32x32x16_f16(p[1], q[0], d, 0, 0, 0);
        d = __builtin_amdgcn_mfma_f32_32x32x16_f16(p[0], q[1], d, 0, 0, 0);
        d = __builtin_amdgcn_mfma_f32_32x32x16_f16(p[0], q[0], d, 0, 0, 0);
      }
      const float f = cc * (sb / (sa * sa)), g = cb * (sb / sa);
#pragma unroll
      for (int e = 0; e < 16; ++e) a[e] = fmaf(f, d[e], g * a[e]);
      put_tile(bm, a, ti, tj);
    }
    __syncthreads();
    // X <- a X + B X
    const float inv = 1.0f / sb, out = 1.0f / sx;
    const bool last = step + 1 == steps;
#pragma unroll
    for (int b = 0; b < SMALL_NB; ++b) {
      if (b >= nb) continue;
      f32x16 d[RB] = {};
#pragma unroll
      for (int r = 0; r < RB; ++r)
#pragma unroll
        for (int c = 0; c < 2 * RB; ++c) {
          half8 p[2];
#pragma unroll
          for (int h = 0; h < 2; ++h) p[h] = rows_of(bm, r, c, h);
          d[r] = __builtin_amdgcn_mfma_f32_32x32x16_f16(p[1], __builtin_bit_cast(half8, x[b][c >> 1][c & 1][0]), d[r], 0, 0, 0);
          d[r] = __builtin_amdgcn_mfma_f32_32x32x16_f16(p[0], __builtin_bit_cast(half8, x[b][c >> 1][c & 1][1]), d[r], 0, 0, 0);
          d[r] = __builtin_amdgcn_mfma_f32_32x32x16_f16(p[0], __builtin_bit_cast(half8, x[b][c >> 1][c & 1][0]), d[r], 0, 0, 0);
        }
#pragma unroll
      for (int r = 0; r < RB; ++r) {
        float v[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          auto half_at = [&](int h) {
            const uint32_t word = x[b][r][e >> 3][h][(e & 7) >> 1];  // (a bit cast of the vector's element itself reads element 0)
            return (float)__builtin_bit_cast(half2_, word)[e & 1];
          };
          v[e] = fmaf(ca, half_at(0) + half_at(1), d[r][e] * inv);
        }
        if (!last) {
#pragma unroll
          for (int e = 0; e < 16; e += 2) keep(x[b][r], e, v[e], v[e + 1]);
        } else {
          int row4 = hf * 4, col = l32;
          asm volatile("" : "+v"(row4), "+v"(col));  // (addresses made here, not kept through the steps)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int j = (wave + 8 * b) * 32 + col, i = r * 32 + (e >> 2) * 8 + row4 + (e & 3);
            if (j < L && i < S) from_f32(v[e] * out, ((E *)m.out)[(uint32_t)(tall ? j * S + i : i * L + j)]);
          }
        }
        packed(x[b][r]);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  }
}

static bool is_small(int rows, int cols) {
  const int s = rows < cols ? rows : cols, l = rows < cols ? cols : rows;
  return s <= SMALL_S && l <= SMALL_L;
}

// f16 halves a factor is held in.  bf16 matrices with a short side beyond 64 make do with one: the errors of 11-bit factors, beside the 8-bit result's own
// rounding of 1.66e-3 (relative, Frobenius), come to 2.0e-3 .. 2.8e-3 in all (4096 x 4096 1.98e-3; short sides of 80 to 200 the most).  On short sides
// of 64 and less there are too few directions for them to average out (64 x 576 4.1e-3, 1 x 7 6.3e-3), and a second half costs little (64 x 576 alone
// 34 -> 55 us; 1536 x 1536 would take 480 instead of 260).
static int planes_of(int32_t dtype, int rows, int cols) { return dtype == AZ_NN_BF16 && (rows < cols ? rows : cols) > SMALL_S ? 1 : 2; }

static int64_t round_up(int64_t v) { return (v + 255) / 256 * 256; }

// tile side by the short side: measured on 1536 x 1536 / 2000 x 4096, 64 takes 0.47 / 1.54 ms in f32 and 0.25 / 0.76 ms in bf16, 128 takes
// 0.53 / 1.34 and 0.34 / 0.59
static int tile_of(int rows, int cols) { return (rows < cols ? rows : cols) >= 1792 ? 128 : 64; }

static bool in_class(int32_t dtype, int rows, int cols, int planes, int tile) {
  return rows > 0 && cols > 0 && planes_of(dtype, rows, cols) == planes && tile_of(rows, cols) == tile;
}

// One workgroup a matrix where every matrix that would share the launches of the others (two halves, tiles of 64) is small; beside larger ones
// they cost nothing in those launches, and a launch of their own would (64 x 576 f32 alone: 88 us in 17 launches, 54 in one).
static bool all_small(int32_t dtype, int count, const int32_t *rows, const int32_t *cols) {
  for (int i = 0; i < count; ++i)
    if (in_class(dtype, rows[i], cols[i], 2, 64) && !is_small(rows[i], cols[i])) return false;
  return true;
}

static int check(const char *&msg, int32_t dtype, int32_t count, const int32_t *rows, const int32_t *cols) {
  if (dtype != AZ_NN_F32 && dtype != AZ_NN_BF16 && dtype != AZ_NN_F16) { msg = "orthogonalize: unknown dtype"; return AZ_EINVAL; }
  if (count < 0 || (count > 0 && (!rows || !cols))) { msg = "orthogonalize: count >= 0, rows and cols given"; return AZ_EINVAL; }
  for (int i = 0; i < count; ++i)
    if (rows[i] < 0 || cols[i] < 0 || rows[i] > 65536 || cols[i] > 65536) { msg = "orthogonalize: sides of 0 .. 65,536"; return AZ_EINVAL; }
  return AZ_OK;
}

// Singular values stay in [0, top]: top of step k + 1 is the largest |a s + b s^3 + c s^5| over [0, top of step k].  The stored X, A and
// B are f16, so coefficients that let them grow without bound are refused.  -> the scales under which entries (at most the largest
// singular value, its square, and the largest |b s^2 + c s^4|) stay below 2^15, half of f16's range
static bool bounded(int steps, double a, double b, double c, Args &g) {
  if (!std::isfinite(a) || !std::isfinite(b) || !std::isfinite(c)) return false;
  double top = 1.0, most = 1.0, poly = 0.0;
  for (int k = 0; k < steps; ++k) {
    double next = 0.0;
    for (int i = 0; i <= 512; ++i) {
      const double s = top * i / 512.0, s2 = s * s;
      next = std::fmax(next, std::fabs(s * (a + s2 * (b + c * s2))));
      poly = std::fmax(poly, std::fabs(s2 * (b + c * s2)));
    }
    if (!(poly < 100.0) || !(next < 7.5)) return false;
    top = next * 1.001;
    most = std::fmax(most, top);
  }
  auto scale = [](double largest) { return (float)std::exp2(std::floor(std::log2(32768.0 / std::fmax(largest, 1.0)))); };
  g.sx = scale(most);
  g.sa = scale(most * most);
  g.sb = scale(poly);
  return true;
}

// One run of launches: up to MAX_M matrices of one tile size and number of halves, and where everything lies in the workspace.
struct Run {
  Table t;
  int planes, tile;
  uint32_t n[6];
  uint64_t part, bytes;
};

// f(Run &) for every run of the call but the small matrices' where k_os_small takes those; in / out may be null (sizes only)
template <class F> static int each_run(int32_t dtype, int count, const void *const *in, void *const *out, const int32_t *rows, const int32_t *cols, F f) {
  const bool small = all_small(dtype, count, rows, cols);
  for (int kind = small ? 1 : 0; kind < 4; ++kind) {
    const int planes = kind < 2 ? 2 : 1, tile = kind & 1 ? 128 : 64;
    Run r;
    r.t.count = 0;
    for (int i = 0; i < count; ++i) {
      if (in_class(dtype, rows[i], cols[i], planes, tile)) {
        r.t.m[r.t.count++] = Mat{in ? in[i] : nullptr, out ? out[i] : nullptr, 0, rows[i], cols[i]};
      }
      if (r.t.count == 0 || (r.t.count < MAX_M && i < count - 1)) continue;
      uint64_t off = round_up(sizeof(Table));
      r.planes = planes;
      r.tile = tile;
      for (uint32_t &v : r.n) v = 0;
      for (int k = 0; k < r.t.count; ++k) {
        Mat &m = r.t.m[k];
        const Lay y(m.rows, m.cols, planes, tile);
        m.ws = off;
        off += (uint64_t)round_up(y.bytes());
        const Split split = split_of(y, tile);
        const int sym = tiles_of<GRAM>(y, tile), cut = sym - split.whole;
        r.t.shares[k] = split.shares;
        const uint32_t add[6] = {(uint32_t)sym, (uint32_t)tiles_of<UPDATE>(y, tile), (uint32_t)(y.sp / 64) * (uint32_t)(y.lp / 64),
                                 (uint32_t)(cut * split.shares), (uint32_t)cut, (uint32_t)split.whole};
        for (int q = 0; q < 6; ++q) { r.t.start[q][k] = r.n[q]; r.n[q] += add[q]; }
      }
      r.part = off;
      off += (uint64_t)r.n[3] * tile * tile * 4;
      r.bytes = off;
      const int rc = f(r);
      if (rc != AZ_OK) return rc;
      r.t.count = 0;
    }
  }
  return AZ_OK;
}

template <class E> static int run_small(const Args &a, int steps, int count, const void *const *in, void *const *out, const int32_t *rows, const int32_t *cols, hipStream_t s) {
  for (int rb = 1; rb <= 2; ++rb) {
    SmallTable t;
    int n = 0;
    for (int i = 0; i < count; ++i) {
      const int side = rows[i] < cols[i] ? rows[i] : cols[i];
      if (side > 0 && is_small(rows[i], cols[i]) && (side <= 32) == (rb == 1)) t.m[n++] = Mat{in[i], out[i], 0, rows[i], cols[i]};
      if (n == 0 || (n < MAX_M && i < count - 1)) continue;
      if (rb == 1) hipLaunchKernelGGL((k_os_small<E, 1>), dim3(n), dim3(SMALL_NT), 0, s, t, a.a, a.b, a.c, a.eps, a.sx, a.sa, a.sb, steps);
      else hipLaunchKernelGGL((k_os_small<E, 2>), dim3(n), dim3(SMALL_NT), 0, s, t, a.a, a.b, a.c, a.eps, a.sx, a.sa, a.sb, steps);
      n = 0;
    }
  }
  return launched("k_os_small");
}

template <class E, int P, int T> static int run(const Run &r, Args a, int steps, hipStream_t s) {
  int parts = 1;
  for (int i = 0; i < r.t.count; ++i) {
    const int own = parts_of(r.t.m[i].rows, r.t.m[i].cols);
    parts = own > parts ? own : parts;
  }
  a.count = r.t.count;
  a.part = r.part;
  for (int k = 0; k < 6; ++k) a.n[k] = (int)r.n[k];
  const dim3 sym(grid_of(r.n[0])), all(grid_of(r.n[1])), split(grid_of(r.n[5]) + grid_of(r.n[3])), join(grid_of(r.n[4]));
  hipLaunchKernelGGL((k_os_norm<E>), dim3(parts, r.t.count), dim3(NT), 0, s, r.t, a.ws);
  hipLaunchKernelGGL((k_os_pack<E, P, T>), dim3(grid_of(r.n[2])), dim3(NT), 0, s, a);
  for (int k = 0; k < steps; ++k) {
    a.cur = k & 1;
    if (r.n[3]) {
      hipLaunchKernelGGL((k_os_gemm<GRAM, P, T, E, SPLIT>), split, dim3(NT), 0, s, a);
      hipLaunchKernelGGL((k_os_gemm<GRAM, P, T, E, JOIN>), join, dim3(NT), 0, s, a);
    } else {
      hipLaunchKernelGGL((k_os_gemm<GRAM, P, T, E, WHOLE>), sym, dim3(NT), 0, s, a);
    }
    if (T == 128 && r.n[3]) {
      if constexpr (T == 128) {
        hipLaunchKernelGGL((k_os_gemm<POLY, P, T, E, SPLIT>), split, dim3(NT), 0, s, a);
        hipLaunchKernelGGL((k_os_gemm<POLY, P, T, E, JOIN>), join, dim3(NT), 0, s, a);
      }
    } else {
      hipLaunchKernelGGL((k_os_gemm<POLY, P, T, E, WHOLE>), sym, dim3(NT), 0, s, a);
    }
    if (k + 1 < steps) hipLaunchKernelGGL((k_os_gemm<UPDATE, P, T, E, WHOLE>), all, dim3(NT), 0, s, a);
    else hipLaunchKernelGGL((k_os_gemm<LAST, P, T, E, WHOLE>), all, dim3(NT), 0, s, a);
  }
  return launched("k_os");
}

}  // namespace azortho

extern "C" {

int64_t az_orthogonalize_workspace(int32_t dtype, int32_t count, const int32_t *rows, const int32_t *cols) {
  using namespace azortho;
  const char *msg = "";
  if (check(msg, dtype, count, rows, cols) != AZ_OK) { fail(AZ_EINVAL, msg); return -1; }
  uint64_t most = 0;  // (runs follow each other on the stream: they share the memory)
  each_run(dtype, count, nullptr, nullptr, rows, cols, [&](const Run &r) {
    most = r.bytes > most ? r.bytes : most;
    return AZ_OK;
  });
  return (int64_t)most;
}

int az_orthogonalize(int32_t dtype, int32_t count, const void *const *in, void *const *out, const int32_t *rows, const int32_t *cols,
                     int32_t steps, double a, double b, double c, double eps, void *workspace_dev, int64_t workspace_bytes, void *stream) {
  using namespace azortho;
  const char *msg = "";
  if (check(msg, dtype, count, rows, cols) != AZ_OK) return fail(AZ_EINVAL, msg);
  if (steps < 1 || steps > 64) return fail(AZ_EINVAL, "orthogonalize: 1 .. 64 steps");
  if (!(eps >= 0.0 && eps < 1e300)) return fail(AZ_EINVAL, "orthogonalize: eps >= 0");
  Args g{};
  if (!bounded(steps, a, b, c, g)) return fail(AZ_EINVAL, "orthogonalize: these coefficients let singular values grow beyond 7.5 (or the polynomial beyond 100)");
  const int es = dtype == AZ_NN_F32 ? 4 : 2;
  if (count > 0 && (!in || !out)) return fail(AZ_EINVAL, "orthogonalize: null argument");
  int live = 0;
  for (int i = 0; i < count; ++i) {
    if (rows[i] == 0 || cols[i] == 0) continue;
    ++live;
    if (!in[i] || !out[i] || misaligned(in[i], es) || misaligned(out[i], es)) return fail(AZ_EINVAL, "orthogonalize: null or misaligned matrix");
  }
  if (live == 0) return AZ_OK;
  const int64_t need = az_orthogonalize_workspace(dtype, count, rows, cols);
  if (need > 0 && (!workspace_dev || misaligned(workspace_dev, 256) || workspace_bytes < need))
    return fail(AZ_EINVAL, "orthogonalize: workspace below az_orthogonalize_workspace() or not aligned to 256 bytes");
  hipStream_t s = (hipStream_t)stream;
  DeviceGuard guard(s);
  if (!guard.ok) return fail(AZ_EHIP, "orthogonalize: cannot select the stream's device");
  g.ws = (char *)workspace_dev;
  g.a = (float)a; g.b = (float)b; g.c = (float)c; g.eps = eps;
  if (all_small(dtype, count, rows, cols)) {
    const int rc = dtype == AZ_NN_F32 ? run_small<float>(g, steps, count, in, out, rows, cols, s) : dtype == AZ_NN_BF16 ? run_small<bf16_t>(g, steps, count, in, out, rows, cols, s)
                                                                                                                : run_small<f16_t>(g, steps, count, in, out, rows, cols, s);
    if (rc != AZ_OK) return rc;
  }
  return each_run(dtype, count, in, out, rows, cols, [&](const Run &r) {
    if (r.planes == 1) return r.tile == 64 ? run<bf16_t, 1, 64>(r, g, steps, s) : run<bf16_t, 1, 128>(r, g, steps, s);
    if (r.tile == 64) return dtype == AZ_NN_F32 ? run<float, 2, 64>(r, g, steps, s) : dtype == AZ_NN_BF16 ? run<bf16_t, 2, 64>(r, g, steps, s) : run<f16_t, 2, 64>(r, g, steps, s);
    return dtype == AZ_NN_F32 ? run<float, 2, 128>(r, g, steps, s) : run<f16_t, 2, 128>(r, g, steps, s);
  });
}

}  // extern "C"
