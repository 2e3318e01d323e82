// Orthogonalisation of matrix updates (the LoRA factors') by Newton-Schulz products:
//   X0 = G / (|G|_F + eps),   X <- P X  with  P = a I + b A + c A^2,  A = X X^T   (steps times)
// With the short side r as rows, every P is a polynomial of A0 = X0 X0^T, so the P commute and are symmetric: the products
// run on r x r matrices alone,  A <- P A P,  Q <- P Q,  and the result is  Q G  (Q starts as I / (|G|_F + eps)): G is read
// for A0 and for the last product.
//
// A and Q are kept and multiplied in 64 bits (v_mfma_f64_16x16x4_f64). A holds the squares of the singular values: in 32
// bits those under 2^-12 of the largest would drown in A's rounding, and the products blow such a value up by a = 3.4
// each step (its square's error by a^2); in 64 bits the result is that of the formula to fp32's own rounding. The sums
// of A0 run in 64 bits for the same reason; products of fp32 values are exact there.
//
// That growth bounds the steps of a pass. A singular value of zero is +-2^-53 in A0; a^(2 k) of it after k steps, and once a
// negative one reaches about -1, P grows without end there (X X^T formed anew has no negative eigenvalues). So a pass takes K steps
// with a^(2 K) <= 2^24 (6 of the usual coefficients: A is right to 2^-29 still); to 2 K steps run as two passes, X between them
// in 64 bits; more as the formula itself on X in 64 bits, X <- a X + (b A + c A^2) X, A formed in each: null directions then
// carry what the formula's own rounding leaves in them, and equal rows stay equal.
//
// The accumulator layout of the f64 instruction (register m of lane l: row 4 m + l / 16, column l % 16) is its layout of
// the operand B at step m of a 16-long contraction, and of the operand A of a symmetric matrix: results are the next
// product's operands as they are.
//
// Kernels: gram (a block per part of a matrix's columns: the part's upper tiles of A0), then for r <= 32 apply with the steps
// inside (every block of a matrix runs them again: two launches in all), for r <= 64 iterate (a block per matrix) and apply,
// and above that the products as launches of their own, a wave per tile (a block per matrix would leave most CUs idle: 128 x 128
// products of 17 cost 130 us of one CU's matrix units). Nothing is atomic: results repeat bit for bit.
#include <stddef.h>

#include <algorithm>
#include <utility>

#include "../../include/smel_ortho.h"
#include "abi_util.h"
#include "common.h"

namespace {

typedef double f64x4_t __attribute__((ext_vector_type(4)));
SMEL_DEV f64x4_t mfma64(double a, double b, f64x4_t c) { return __builtin_amdgcn_mfma_f64_16x16x4f64(a, b, c, 0, 0, 0); }

// the binding packs a job as nine 8-byte values in this order
static_assert(sizeof(smel_ortho_job) == 72 && offsetof(smel_ortho_job, x) == 0 && offsetof(smel_ortho_job, y) == 8 &&
                  offsetof(smel_ortho_job, batch) == 16 && offsetof(smel_ortho_job, rows) == 24 && offsetof(smel_ortho_job, cols) == 32 &&
                  offsetof(smel_ortho_job, x_batch) == 40 && offsetof(smel_ortho_job, x_row) == 48 &&
                  offsetof(smel_ortho_job, x_col) == 56 && offsetof(smel_ortho_job, dtype) == 64,
              "layout of a job");

constexpr int MAX_R = 128;
constexpr int MAX_JOBS = 36;   // of one launch: the jobs travel as kernel arguments (under 4 KiB)
constexpr int WAVES = 8;       // of a gram or apply block

struct Job {
  const void* x;
  void* y;
  int64_t xb, ld;      // batch stride; stride between lines (a line: the side with unit stride)
  int64_t part0;       // first tile-set slot of the job's parts in the workspace
  int32_t batch, r, n;
  int32_t blk0, mat0;  // first block (gram, apply) and first matrix (iterate, Q)
  int32_t slices;      // of a matrix
  int32_t gblk0, parts;   // gram: first block, blocks of a matrix (each takes js.per columns)
  int32_t x_tall;      // 1: the short side has the unit stride in x
  int32_t y_tall;      // 1: the short side is y's last
};
struct Jobs {
  int32_t n, lg;      // jobs; log2 of the columns of an apply block's slice (64 at least)
  int32_t glg, per;   // log2 of the columns of a gram slice; columns of a gram block, a multiple of 16
  Job j[MAX_JOBS];
};
static_assert(sizeof(Jobs) <= 3584, "kernel arguments");

constexpr int ntiles(int nt) { return nt * (nt + 1) / 2; }
// upper tile k -> (t, u), t <= u, row by row
SMEL_DEV void tile_of(int k, int nt, int& t, int& u) {
  t = 0;
  while (k >= nt - t) {
    k -= nt - t;
    ++t;
  }
  u = t + k;
}
SMEL_DEV int tile_at(int t, int u, int nt) { return t * nt - t * (t - 1) / 2 + (u - t); }   // t <= u

template <int DT>
SMEL_DEV float to_f(uint32_t b) {
  if constexpr (DT == 0) return __uint_as_float(b << 16);
  return (float)__builtin_bit_cast(_Float16, (uint16_t)b);
}
template <int DT>
struct Elem {
  typedef uint16_t T;
};
template <>
struct Elem<1> {
  typedef float T;
};
// the job of block (gram, apply) or matrix b; uniform
enum { BY_GRAM, BY_APPLY, BY_MATRIX };
template <int BY>
SMEL_DEV int find_job(const Jobs& js, int b) {
  int k = 0;
  while (k + 1 < js.n && b >= (BY == BY_GRAM ? js.j[k + 1].gblk0 : BY == BY_APPLY ? js.j[k + 1].blk0 : js.j[k + 1].mat0)) ++k;
  return k;
}

typedef u32x4_t __attribute__((aligned(2))) u32x4_a2;
typedef f32x4_t __attribute__((aligned(4))) f32x4_a4;
typedef uint32_t __attribute__((ext_vector_type(2), aligned(2))) u32x2_a2;
// N (4 or 8) consecutive floats, `left` of them in range: 16-byte stores at any alignment
template <int N>
SMEL_DEV void st_run(float* p, int left, const double* v) {
  if (left >= N) {
#pragma unroll
    for (int k = 0; k < N; k += 4) *(f32x4_a4*)(p + k) = f32x4_t{(float)v[k], (float)v[k + 1], (float)v[k + 2], (float)v[k + 3]};
    return;
  }
#pragma unroll
  for (int k = 0; k < N; ++k)
    if (k < left) p[k] = (float)v[k];
}

template <int DT>
struct Vec {
  static constexpr int V = DT == 1 ? 4 : 8;   // elements of 16 bytes
};
// V consecutive elements as stored (16 bytes), zeros past `left`; 16-byte loads at any alignment
template <int DT>
SMEL_DEV u32x4_t ld_raw(const typename Elem<DT>::T* p, int left) {
  constexpr int V = Vec<DT>::V;
  if (left >= V) {
    if constexpr (DT == 1)
      return __builtin_bit_cast(u32x4_t, (f32x4_t)*(const f32x4_a4*)p);
    else
      return *(const u32x4_a2*)p;
  }
  if (left <= 0) return u32x4_t{0, 0, 0, 0};
  uint32_t v[V];
#pragma unroll
  for (int k = 0; k < V; ++k) {
    const auto e = p[min(k, left - 1)];   // in range; dropped past it
    if constexpr (DT == 1)
      v[k] = k < left ? __float_as_uint(e) : 0u;
    else
      v[k] = k < left ? (uint32_t)e : 0u;
  }
  if constexpr (DT == 1)
    return u32x4_t{v[0], v[1], v[2], v[3]};
  else
    return u32x4_t{v[0] | v[1] << 16, v[2] | v[3] << 16, v[4] | v[5] << 16, v[6] | v[7] << 16};
}
template <int DT>
SMEL_DEV float raw_at(const u32x4_t& r, int k) {
  if constexpr (DT == 1)
    return __uint_as_float(r[k]);
  else
    return to_f<DT>((k & 1) ? r[k >> 1] >> 16 : r[k >> 1] & 0xffffu);
}

// Columns [j0, j0 + slice) of a matrix on the way to LDS, where they lie as fp32 X[i][j], rows [r, 16 NT) and columns past n
// zero: fetch issues the loads, put converts and writes. W waves; slice <= S. The pitch of slice + 20 floats (20 mod 64
// banks) keeps the 16 rows of a gram operand and the 16 columns x 4 chunks of a transposed store apart.
template <int NT, int DT, int W, int S>
struct Slice {
  static constexpr int V = Vec<DT>::V, RP = 16 * NT, CH = (RP * S / V + 64 * W - 1) / (64 * W);
  static constexpr int LV = V == 4 ? 2 : 3;
  u32x4_t raw[CH];

  // row and column of chunk e (lines along i: 16 lanes take a chunk of 16 lines)
  SMEL_DEV static int row(bool tall, int e, int lg) { return tall ? (e >> 4) % (RP / V) * V : e >> (lg - LV); }
  SMEL_DEV static int col(bool tall, int e, int lg) { return tall ? e / (16 * RP / V) * 16 + (e & 15) : (e << LV) & ((1 << lg) - 1); }
  SMEL_DEV void fetch(const Job& J, int mat, int j0, int end, int lg) {
    const int slice = 1 << lg;
    typedef typename Elem<DT>::T T;
    const T* const x = (const T*)J.x + mat * J.xb;
    const int nc = min(slice, end - j0);
#pragma unroll
    for (int q = 0; q < CH; ++q) {
      const int e = threadIdx.x + q * 64 * W;
      const int i = row(J.x_tall, e, lg), j = col(J.x_tall, e, lg);
      if (e >= (RP << lg) / V) continue;
      if (J.x_tall)
        raw[q] = ld_raw<DT>(x + (int64_t)(j0 + j) * J.ld + i, j < nc ? J.r - i : 0);
      else
        raw[q] = ld_raw<DT>(x + i * J.ld + j0 + j, i < J.r ? nc - j : 0);
    }
  }
  SMEL_DEV void put(bool tall, int lg, float* X, int pitch) const {
#pragma unroll
    for (int q = 0; q < CH; ++q) {
      const int e = threadIdx.x + q * 64 * W;
      const int i = row(tall, e, lg), j = col(tall, e, lg);
      if (e >= (RP << lg) / V) continue;
      if (tall) {
#pragma unroll
        for (int k = 0; k < V; ++k) X[(i + k) * pitch + j] = raw_at<DT>(raw[q], k);
      } else {
#pragma unroll
        for (int k = 0; k < V; k += 4)
          *(f32x4_t*)(X + i * pitch + j + k) = f32x4_t{raw_at<DT>(raw[q], k), raw_at<DT>(raw[q], k + 1), raw_at<DT>(raw[q], k + 2),
                                                       raw_at<DT>(raw[q], k + 3)};
      }
    }
  }
};

// columns of an apply block's slice at most: two blocks on a CU
constexpr int max_slice(int nt) { return nt == 1 ? 1024 : nt <= 4 ? 256 : 128; }
constexpr int max_slice16(int nt) { return nt == 1 ? 1024 : nt == 2 ? 512 : nt == 4 ? 256 : 128; }   // of 16-bit types

// A gram block takes `per` columns in slices, the next one on its way while one is multiplied (two buffers). Waves of a block: the
// upper tiles in TG groups, a group's columns dealt to the others. Three tiles a wave at r = 128: nine leave registers for two
// waves a SIMD, too few to cover the operands' latencies (36 x 128 x 2816: 65 us, three: 55; one round of blocks with the
// loads ahead: see the plan's `per`; blocks of 416 columns, not of 448 in whole slices: 43 -> 41.6).
constexpr int gram_slice(int nt) { return nt == 1 ? 512 : nt == 2 ? 256 : nt == 4 ? 128 : 64; }
constexpr int gram_waves(int nt) { return nt == 8 ? 12 : WAVES; }
constexpr int gram_tg(int nt) { return nt == 8 ? 12 : nt == 4 ? 2 : 1; }
// At r = 128 a wave's three tiles share their operands: the 28 pairs of eight rows of tiles are eight triangles (the lines of the
// affine plane of order 3 that miss a point: rows a, b, c give the tiles ab, ac, bc) and four pairs left over, each with its
// rows' diagonal tiles. Half the LDS reads and conversions of three tiles of their own (36 x 128 x 2816: 50 -> 43 us).
constexpr uint16_t GRAM_ROWS[12] = {0x012, 0x345, 0x036, 0x147, 0x156, 0x237, 0x057, 0x246, 0x677, 0x255, 0x044, 0x133};

template <int NT, int DT>
__global__ __launch_bounds__(64 * gram_waves(NT)) void gram_kernel(Jobs js, double* __restrict__ part) {
  constexpr int NTL = ntiles(NT), W = gram_waves(NT), TG = gram_tg(NT), KG = W / TG, TPW = NTL / TG;
  constexpr int S = gram_slice(NT), BUF = 16 * NT * (S + 20);
  static_assert(TPW * TG == NTL && KG * TG == W, "tiles per wave");
  static_assert(2 * BUF * 4 >= NTL * 2048 || KG == 1, "room for the column groups' sums");
  __shared__ __attribute__((aligned(16))) float X[2 * BUF];
  const int lg = js.glg, slice = 1 << lg, pitch = slice + 20;
  const Job& J = js.j[find_job<BY_GRAM>(js, blockIdx.x)];
  const int lb = blockIdx.x - J.gblk0, mat = lb / J.parts, c1 = min((lb % J.parts + 1) * js.per, J.n);
  int c0 = lb % J.parts * js.per;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, lo = lane & 15, hi = lane >> 4;
  const int tg = wave % TG, kg = wave / TG;
  f64x4_t acc[TPW];
  int ra[TPW], rb[TPW], tile[TPW];
  const uint32_t rows = GRAM_ROWS[wave % 12];
  const bool triangle = wave < 8;
#pragma unroll
  for (int k = 0; k < TPW; ++k) {
    acc[k] = f64x4_t{0, 0, 0, 0};
    int t, u;
    if constexpr (NT == 8) {   // ra: the three rows' operands
      const int r[3] = {(int)(rows >> 8), (int)(rows >> 4 & 15), (int)(rows & 15)};
      ra[k] = (16 * r[k] + lo) * pitch + 4 * hi;
      t = r[k == 2];
      u = triangle ? r[k == 0 ? 1 : 2] : r[k == 0 || k == 2];
    } else {
      tile_of(tg * TPW + k, NT, t, u);
      ra[k] = (16 * t + lo) * pitch + 4 * hi;
      rb[k] = (16 * u + lo) * pitch + 4 * hi;
    }
    tile[k] = tile_at(t, u, NT);
  }
  Slice<NT, DT, W, S> in;
  in.fetch(J, mat, c0, c1, lg);
  in.put(J.x_tall, lg, X, pitch);
  __syncthreads();
  for (int buf = 0; c0 < c1; c0 += slice, buf ^= 1) {
    const float* const x = X + buf * BUF;
    const bool more = c0 + slice < c1;
    const int width = min(slice, c1 - c0);
    if (more) in.fetch(J, mat, c0 + slice, c1, lg);
    // 16 columns a step, four to a lane: which columns make one instruction's contraction does not matter
    if constexpr (NT == 8) {
      for (int j = 0; j < width; j += 16) {
        const f32x4_t a = *(const f32x4_t*)(x + ra[0] + j), b = *(const f32x4_t*)(x + ra[1] + j);
        if (triangle) {
          const f32x4_t c = *(const f32x4_t*)(x + ra[2] + j);
#pragma unroll
          for (int m = 0; m < 4; ++m) {
            const double am = a[m], bm = b[m], cm = c[m];
            acc[0] = mfma64(am, bm, acc[0]);
            acc[1] = mfma64(am, cm, acc[1]);
            acc[2] = mfma64(bm, cm, acc[2]);
          }
        } else {
#pragma unroll
          for (int m = 0; m < 4; ++m) {
            const double am = a[m], bm = b[m];
            acc[0] = mfma64(am, bm, acc[0]);
            acc[1] = mfma64(am, am, acc[1]);
            acc[2] = mfma64(bm, bm, acc[2]);
          }
        }
      }
    } else {
      for (int j = 16 * kg; j < width; j += 16 * KG)
#pragma unroll
        for (int k = 0; k < TPW; ++k) {
          const f32x4_t a = *(const f32x4_t*)(x + ra[k] + j), b = *(const f32x4_t*)(x + rb[k] + j);
#pragma unroll
          for (int m = 0; m < 4; ++m) acc[k] = mfma64(a[m], b[m], acc[k]);
        }
    }
    if (more) in.put(J.x_tall, lg, X + (buf ^ 1) * BUF, pitch);
    __syncthreads();
  }
  // the column groups' sums, in group order
  f64x4_t* const red = (f64x4_t*)X;   // [TG][TPW][64]
  double* const out = part + (J.part0 + lb) * (int64_t)(NTL * 256);
  for (int g = 1; g < KG; ++g) {
    if (g > 1) __syncthreads();
    if (kg == g)
#pragma unroll
      for (int k = 0; k < TPW; ++k) red[(tg * TPW + k) * 64 + lane] = acc[k];
    __syncthreads();
    if (kg == 0)
#pragma unroll
      for (int k = 0; k < TPW; ++k) acc[k] += red[(tg * TPW + k) * 64 + lane];
  }
  if (kg == 0)
#pragma unroll
    for (int k = 0; k < TPW; ++k) *(f64x4_t*)(out + (tile[k] * 64 + lane) * 4) = acc[k];
}

struct Steps {
  int32_t steps;
  int32_t normed;   // 1: the matrix is X already, no norm is taken out
  double a, b, c, eps;
};
// 1 / (|G|_F + eps) of a trace of A0
SMEL_DEV double inv_norm(const Steps& st, double trace) { return st.normed ? 1.0 : 1.0 / (sqrt(trace) + st.eps); }

// Q carries 1 / (|G|_F + eps) = s. Outside 2^-64 to 2^64 (an update of tiny norm with eps near 0, or of values near the type's
// largest, whose s would leave its second and third bf16 part under their smallest value) a power of two stays out of it, so
// that Q's bf16 parts stay in range; the last product multiplies it back in. exp_of(s): that power's exponent.
SMEL_DEV int exp_of(double s) {
  if (s > 0x1p64 && s < 0x1p1000) return ilogb(s) - 64;
  return s < 0x1p-64 && s > 0x1p-1000 ? ilogb(s) + 64 : 0;
}

constexpr int TP = 17;   // doubles between the rows of a tile in LDS

constexpr int IT_WAVES = 10;   // of an iterate block: an upper tile each (r <= 64)

// element (16 u + 4 m + l / 16, 16 t + l % 16) of a symmetric matrix in upper tiles: at + m * step
SMEL_DEV int frag_at(int u, int t, int nt, int lo, int hi, int& step) {
  if (u <= t) {
    step = 4 * TP;
    return tile_at(u, t, nt) * (16 * TP) + hi * TP + lo;
  }
  step = 4;
  return tile_at(t, u, nt) * (16 * TP) + lo * TP + hi;
}

// The steps of 32 < r <= 64, a block per matrix and a wave per upper tile; three barriers a step
__global__ __launch_bounds__(64 * IT_WAVES) void iterate_kernel(Jobs js, Steps st, const double* __restrict__ part,
                                                                double* __restrict__ Qout, double* __restrict__ qscale) {
  constexpr int NT = 4, NTL = ntiles(NT), SIZE = NTL * 16 * TP;
  static_assert(NTL == IT_WAVES, "a tile per wave");
  __shared__ double bA[SIZE], bP[SIZE], bT[SIZE], bQ[SIZE], trs[NT];
  const Job& J = js.j[find_job<BY_MATRIX>(js, blockIdx.x)];
  const int mat = blockIdx.x - J.mat0;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, lo = lane & 15, hi = lane >> 4;
  int t, u;
  tile_of(wave, NT, t, u);
  f64x4_t A = {0, 0, 0, 0}, eye;
  const double* const p = part + (J.part0 + (int64_t)mat * J.parts) * (NTL * 256) + (wave * 64 + lane) * 4;
#pragma unroll 8
  for (int s = 0; s < J.parts; ++s) A += *(const f64x4_t*)(p + (int64_t)s * (NTL * 256));
  double d = 0;   // the tile's trace: row 4 m + hi, column lo
#pragma unroll
  for (int m = 0; m < 4; ++m) {
    eye[m] = t == u && 4 * m + hi == lo ? 1.0 : 0.0;
    d += 4 * m + hi == lo ? A[m] : 0.0;
  }
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) d += __shfl_xor(d, o, 64);
  if (t == u && lane == 0) trs[t] = d;
  __syncthreads();
  const double s = inv_norm(st, ((trs[0] + trs[1]) + trs[2]) + trs[3]);
  const double sq = ldexp(s, -exp_of(s));
  if (threadIdx.x == 0) qscale[blockIdx.x] = ldexp(1.0, exp_of(s));
  A = A * s * s;
  f64x4_t Q = eye * sq;
  auto put = [&](double* buf, f64x4_t M) {
#pragma unroll
    for (int m = 0; m < 4; ++m) buf[wave * (16 * TP) + (4 * m + hi) * TP + lo] = M[m];
  };
  auto product = [&](const double* M, const double* N) {
    f64x4_t acc = {0, 0, 0, 0};
#pragma unroll
    for (int k = 0; k < NT; ++k) {
      int sa, sb;
      const int a = frag_at(k, t, NT, lo, hi, sa), b = frag_at(k, u, NT, lo, hi, sb);
#pragma unroll
      for (int m = 0; m < 4; ++m) acc = mfma64(M[a + m * sa], N[b + m * sb], acc);
    }
    return acc;
  };
  for (int it = 0; it < st.steps; ++it) {
    const bool last = it + 1 == st.steps;
    put(bA, A);
    lds_barrier();
    const f64x4_t P = st.b * A + st.c * product(bA, bA) + st.a * eye;
    put(bP, P);
    put(bQ, Q);
    lds_barrier();
    if (!last) put(bT, product(bA, bP));
    Q = it == 0 ? P * sq : product(bP, bQ);
    lds_barrier();
    if (!last) A = product(bT, bP);
  }
  // Q's tiles, both triangles, in the operand layout: tile (k, t) register m of lane l = Q[16 k + 4 m + hi][16 t + lo]
  put(bQ, Q);
  lds_barrier();
  double* const out = Qout + (int64_t)blockIdx.x * (NT * NT * 256);
  for (int k = wave; k < NT * NT; k += IT_WAVES) {
    int sa;
    const int a = frag_at(k / NT, k % NT, NT, lo, hi, sa);
    f64x4_t q;
#pragma unroll
    for (int m = 0; m < 4; ++m) q[m] = bQ[a + m * sa];
    *(f64x4_t*)(out + (k * 64 + lane) * 4) = q;
  }
}

// ------------------------------------------------------------------------------------------------ steps of r <= 32, in a block

// A0 (scaled) and the steps, wave w < NT^2 holding tile (w / NT, w % NT) of every matrix; Q's tiles to bQ. All waves of the
// block call it; returns the power of two that is not in Q. Tiles lie in LDS as they lie in the registers (64 lanes x 4), which
// is the operand layout.
template <int NT>
SMEL_DEV double steps_small(const Job& J, int mat, const Steps& st, const double* __restrict__ part, f64x4_t (*bA)[64],
                            double* tr) {
  constexpr int NTL = ntiles(NT), N2 = NT * NT;
  f64x4_t(*const bP)[64] = bA + N2, (*const bT)[64] = bA + 2 * N2, (*const bQ)[64] = bA + 3 * N2;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, lo = lane & 15, hi = lane >> 4;
  const bool mine = wave < NT * NT;
  const int t = wave / NT, u = wave % NT;
  f64x4_t A = {0, 0, 0, 0}, Q = {0, 0, 0, 0}, P = {0, 0, 0, 0}, S;
  f64x4_t eye;
#pragma unroll
  for (int m = 0; m < 4; ++m) eye[m] = t == u && 4 * m + hi == lo ? 1.0 : 0.0;
  // the parts' sum: GR groups of waves take every GR-th part of an upper tile each, then the groups in order
  constexpr int GR = NT == 1 ? 4 : 2;
  static_assert(GR * NTL <= 4 * NT * NT && GR * NTL <= WAVES, "slots and waves of the sum");
  if (wave < GR * NTL) {
    const int g = wave / NTL;
    const double* const p = part + (J.part0 + (int64_t)mat * J.parts) * (NTL * 256) + (wave % NTL) * 256 + lane * 4;
#pragma unroll 8
    for (int s = g; s < J.parts; s += GR) A += *(const f64x4_t*)(p + (int64_t)s * (NTL * 256));
    bA[wave][lane] = A;     // bA to bQ are one array
  }
  __syncthreads();
  if (mine) {
    // a lower tile is its mirror's transpose: element (4 m + hi, lo) is register lo / 4 of lane (lo % 4, 4 m + hi)
    const int k = t <= u ? tile_at(t, u, NT) : tile_at(u, t, NT);
    A = f64x4_t{0, 0, 0, 0};
#pragma unroll
    for (int g = 0; g < GR; ++g) {
      const f64x4_t(&q)[64] = bA[g * NTL + k];
      if (t <= u) {
        A += q[lane];
      } else {
#pragma unroll
        for (int m = 0; m < 4; ++m) A[m] += ((const double*)q)[((lo & 3) * 16 + 4 * m + hi) * 4 + (lo >> 2)];
      }
    }
    double d = 0;
#pragma unroll
    for (int m = 0; m < 4; ++m) d += eye[m] != 0 ? A[m] : 0.0;
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) d += __shfl_xor(d, o, 64);
    if (t == u && lane == 0) tr[t] = d;
  }
  __syncthreads();
  double sum = tr[0];
#pragma unroll
  for (int k = 1; k < NT; ++k) sum += tr[k];
  const double s = inv_norm(st, sum);
  const int ex = exp_of(s);
  const double sq = ldexp(s, -ex);
  A = A * s * s;
  Q = eye * sq;
  auto product = [&](f64x4_t (*M)[64], f64x4_t (*N)[64]) {
    f64x4_t acc = {0, 0, 0, 0};
#pragma unroll
    for (int k = 0; k < NT; ++k) {
      const f64x4_t a = M[k * NT + t][lane], b = N[k * NT + u][lane];
#pragma unroll
      for (int m = 0; m < 4; ++m) acc = mfma64(a[m], b[m], acc);
    }
    return acc;
  };
  auto own = [&](f64x4_t a, f64x4_t b) {   // NT = 1: the operands are the wave's own registers
    f64x4_t acc = {0, 0, 0, 0};
#pragma unroll
    for (int m = 0; m < 4; ++m) acc = mfma64(a[m], b[m], acc);
    return acc;
  };
  for (int it = 0; it < st.steps; ++it) {
    const bool first = it == 0, last = it + 1 == st.steps;
    if constexpr (NT == 1) {
      if (mine) {
        P = st.b * A + st.c * own(A, A) + st.a * eye;
        if (!last) S = own(A, P);
        Q = first ? P * sq : own(P, Q);
        if (!last) A = own(S, P);
      }
    } else {
      if (mine) bA[wave][lane] = A;
      lds_barrier();
      if (mine) {
        P = st.b * A + st.c * product(bA, bA) + st.a * eye;
        bP[wave][lane] = P;
        bQ[wave][lane] = Q;
      }
      lds_barrier();
      if (mine) {
        if (!last) bT[wave][lane] = product(bA, bP);
        Q = first ? P * sq : product(bP, bQ);
      }
      lds_barrier();
      if (mine && !last) A = product(bT, bP);
    }
  }
  if (mine) bQ[wave][lane] = Q;
  __syncthreads();
  return ldexp(1.0, ex);
}

// Q G for a slice of fp32. SMALL: the steps run here, from the parts; else Q's tiles are read. A wave owns one tile of rows and every
// CG-th pair of 16-column blocks. The columns of a pair (or, for a result whose short side is last, the rows of a tile) are
// dealt to the instruction's rows so that a lane's registers are neighbours in memory.
template <int NT, bool SMALL>
__global__ __launch_bounds__(64 * WAVES, 4) void apply_kernel(Jobs js, Steps st, const double* __restrict__ in,
                                                        const double* __restrict__ qscale) {
  constexpr int CG = WAVES / NT;
  __shared__ __attribute__((aligned(16))) float X[16 * NT * (max_slice(NT) + 20)];
  const int slice = 1 << js.lg, pitch = slice + 20;
  const Job& J = js.j[find_job<BY_APPLY>(js, blockIdx.x)];
  const int lb = blockIdx.x - J.blk0, mat = lb / J.slices, j0 = (lb % J.slices) << js.lg;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, lo = lane & 15, hi = lane >> 4;
  const int t = wave % NT, cg = wave / NT;
  const int perm = 4 * (lo & 3) + (lo >> 2);   // row 4 m + hi of the result <- index 4 hi + m
  const int qlane = J.y_tall ? hi * 16 + perm : lane;
  {
    Slice<NT, 1, WAVES, max_slice(NT)> in;
    in.fetch(J, mat, j0, J.n, js.lg);
    in.put(J.x_tall, js.lg, X, pitch);
  }
  f64x4_t q[NT];
  double scale;
  if constexpr (SMALL) {
    __shared__ f64x4_t b[4 * NT * NT][64];
    __shared__ double tr[NT];
    scale = steps_small<NT>(J, mat, st, in, b, tr);   // ends with a barrier: X and Q's tiles are there
#pragma unroll
    for (int u = 0; u < NT; ++u) q[u] = b[(3 * NT + u) * NT + t][qlane];
  } else {
#pragma unroll
    for (int u = 0; u < NT; ++u)
      q[u] = *(const f64x4_t*)(in + (int64_t)(J.mat0 + mat) * (NT * NT * 256) + ((u * NT + t) * 64 + qlane) * 4);
    scale = qscale[J.mat0 + mat];
    __syncthreads();
  }
#pragma unroll
  for (int u = 0; u < NT; ++u) q[u] = q[u] * scale;
  const int nc = min(slice, J.n - j0);
  float* const y = (float*)J.y + (int64_t)mat * J.r * J.n;
  if (J.y_tall) {
    for (int j = 16 * cg; j < nc; j += 16 * CG) {
      f64x4_t acc = {0, 0, 0, 0};
#pragma unroll
      for (int u = 0; u < NT; ++u)
#pragma unroll
        for (int m = 0; m < 4; ++m) acc = mfma64(q[u][m], (double)X[(16 * u + 4 * m + hi) * pitch + j + lo], acc);
      const int i = 16 * t + 4 * hi;   // rows i + m, column j + lo
      if (j + lo < nc) st_run<4>(y + (int64_t)(j0 + j + lo) * J.r + i, J.r - i, (const double*)&acc);
    }
  } else {
    for (int j = 32 * cg; j < nc; j += 32 * CG) {
      f64x4_t acc[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
      const int c = j + 8 * (lo & 3) + (lo >> 2);   // the pair: columns 8 hi + m and 8 hi + 4 + m
#pragma unroll
      for (int u = 0; u < NT; ++u)
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          const float* const x = X + (16 * u + 4 * m + hi) * pitch + c;
          acc[0] = mfma64((double)x[0], q[u][m], acc[0]);
          acc[1] = mfma64((double)x[4], q[u][m], acc[1]);
        }
      const int i = 16 * t + lo, k = j + 8 * hi;   // row i, columns k to k + 7
      if (i < J.r) st_run<8>(y + (int64_t)i * J.n + j0 + k, nc - k, (const double*)acc);
    }
  }
}

// The same for 16-bit results, whose rounding (2^-9, 2^-12) leaves room for fp32 sums: Q as three bf16 parts (24 bits), G's
// bf16 values as they are and fp16 values as two bf16 parts, products on the bf16 matrix instruction: 36 x 128 x 2816 bf16 took
// 80 us on the f64 instruction. The parts' products are added in fp32: off by at most 3 r 2^-24 of sum |q| |g|.
// Of a tile's 16 rows (the contraction), lane l / 16 = h takes h, 4 + h, 8 + h and 12 + h: the order in which Q's tiles lie.
// G's slice lies in LDS as words of the rows (i, i + 4): word [8 u + 4 k + h][j], rows 16 u + 8 k + h and + 4. Pitch slice + 36:
// the four words' rows that 64 lanes read at 16 columns take the banks twice at most.
typedef short s16x4_t __attribute__((ext_vector_type(4)));
SMEL_DEV f32x4_t mfma16(u32x2_t a, u32x2_t b, f32x4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s16x4_t, a), __builtin_bit_cast(s16x4_t, b), c, 0, 0, 0);
}
SMEL_DEV f32x4_t mfma16(u32x4_t a, u32x4_t b, f32x4_t c) {   // two tiles' rows at once
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}

template <int NT>
SMEL_DEV void load_pairs(const Job& J, int mat, int j0, int lg, uint32_t* X, int pitch) {
  constexpr int RP = 16 * NT;
  const int slice = 1 << lg;
  const uint16_t* const x = (const uint16_t*)J.x + mat * J.xb;
  const int nc = min(slice, J.n - j0);
  if (J.x_tall) {
    constexpr int Q = RP / 8;
    const int chunks = RP * slice / 8;
#pragma unroll 4
    for (int e = threadIdx.x; e < chunks; e += 64 * WAVES) {
      const int j = e / (16 * Q) * 16 + (e & 15), i = (e >> 4) % Q * 8;
      const u32x4_t v = ld_raw<0>(x + (int64_t)(j0 + j) * J.ld + i, j < nc ? J.r - i : 0);
#pragma unroll
      for (int h = 0; h < 4; ++h)
        X[(i / 2 + h) * pitch + j] = (h & 1) ? v[h >> 1] >> 16 | (v[2 + (h >> 1)] & 0xffff0000u)
                                             : (v[h >> 1] & 0xffffu) | v[2 + (h >> 1)] << 16;
    }
  } else {
    const int chunks = RP / 2 << (lg - 3);
#pragma unroll 2
    for (int e = threadIdx.x; e < chunks; e += 64 * WAVES) {
      const int p = e >> (lg - 3), j = (e << 3) & (slice - 1), i = (p >> 2) * 8 + (p & 3);
      const uint16_t* const row = x + i * J.ld + j0 + j;
      const u32x4_t a = ld_raw<0>(row, i < J.r ? nc - j : 0), b = ld_raw<0>(row + 4 * J.ld, i + 4 < J.r ? nc - j : 0);
      u32x4_t w[2];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        w[k >> 1][2 * (k & 1)] = (a[k] & 0xffffu) | b[k] << 16;
        w[k >> 1][2 * (k & 1) + 1] = a[k] >> 16 | (b[k] & 0xffff0000u);
      }
      *(u32x4_t*)(X + p * pitch + j) = w[0];
      *(u32x4_t*)(X + p * pitch + j + 4) = w[1];
    }
  }
}

template <int DT, int N>
SMEL_DEV void st_run16(uint16_t* p, int left, const float* v) {
  uint32_t w[N / 2];
#pragma unroll
  for (int k = 0; k < N / 2; ++k) {
    if constexpr (DT == 0)
      w[k] = pack2bf(v[2 * k], v[2 * k + 1]);
    else
      w[k] = __builtin_bit_cast(uint16_t, (_Float16)v[2 * k]) | (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)v[2 * k + 1]) << 16;
  }
  if (left >= N) {
    if constexpr (N == 8)
      *(u32x4_a2*)p = u32x4_t{w[0], w[1], w[2], w[3]};
    else
      *(u32x2_a2*)p = u32x2_a2{w[0], w[1]};
    return;
  }
#pragma unroll
  for (int k = 0; k < N; ++k)
    if (k < left) p[k] = (uint16_t)((k & 1) ? w[k >> 1] >> 16 : w[k >> 1]);
}

template <int NT, int DT, bool SMALL>
__global__ __launch_bounds__(64 * WAVES, 4) void apply16_kernel(Jobs js, Steps st, const double* __restrict__ in,
                                                          const double* __restrict__ qscale) {
  constexpr int CG = WAVES / NT;
  __shared__ __attribute__((aligned(16))) uint32_t X[8 * NT * (max_slice16(NT) + 36)];
  const int slice = 1 << js.lg, pitch = slice + 36;
  const Job& J = js.j[find_job<BY_APPLY>(js, blockIdx.x)];
  const int lb = blockIdx.x - J.blk0, mat = lb / J.slices, j0 = (lb % J.slices) << js.lg;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, lo = lane & 15, hi = lane >> 4;
  const int t = wave % NT, cg = wave / NT;
  load_pairs<NT>(J, mat, j0, js.lg, X, pitch);
  constexpr int K2 = NT == 1 ? 1 : 2;   // tiles of an instruction's contraction
  typedef uint32_t word_t __attribute__((ext_vector_type(2 * K2)));
  float scale;
  word_t q[NT / K2][3];   // parts of Q[16 t + lo][16 u + 4 m + hi]
  auto parts = [&](int u, f64x4_t v) {
    float r[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) r[k] = (float)v[k];
#pragma unroll
    for (int p = 0; p < 3; ++p) {
      const uint32_t a = pack2bf(r[0], r[1]), b = pack2bf(r[2], r[3]);
      q[u / K2][p][2 * (u % K2)] = a;
      q[u / K2][p][2 * (u % K2) + 1] = b;
      r[0] -= bf_lo(a);
      r[1] -= bf_hi(a);
      r[2] -= bf_lo(b);
      r[3] -= bf_hi(b);
    }
  };
  if constexpr (SMALL) {
    __shared__ f64x4_t b[4 * NT * NT][64];
    __shared__ double tr[NT];
    scale = (float)steps_small<NT>(J, mat, st, in, b, tr);
#pragma unroll
    for (int u = 0; u < NT; ++u) parts(u, b[(3 * NT + u) * NT + t][lane]);
  } else {
    scale = (float)qscale[J.mat0 + mat];
    const double* const Q = in + (int64_t)(J.mat0 + mat) * (NT * NT * 256);
#pragma unroll
    for (int u = 0; u < NT; ++u) parts(u, *(const f64x4_t*)(Q + ((u * NT + t) * 64 + lane) * 4));
    __syncthreads();
  }
  const int nc = min(slice, J.n - j0);
  uint16_t* const y = (uint16_t*)J.y + (int64_t)mat * J.r * J.n;
  // acc += Q G (or its transpose) over the tiles of instruction v, for column c of the lane
  auto dot = [&](int v, int c, bool tall, f32x4_t acc) {
    word_t g, g2;
#pragma unroll
    for (int k = 0; k < 2 * K2; ++k) {
      const uint32_t w = X[(8 * K2 * v + 4 * k + hi) * pitch + c];
      if constexpr (DT == 0) {
        g[k] = w;
      } else {
        const float f0 = to_f<2>(w & 0xffffu), f1 = to_f<2>(w >> 16);
        g[k] = pack2bf(f0, f1);
        g2[k] = pack2bf(f0 - bf_lo(g[k]), f1 - bf_hi(g[k]));
      }
    }
#pragma unroll
    for (int p = 2; p >= 0; --p) {
      if (DT == 2 && p < 2) acc = tall ? mfma16(q[v][p], g2, acc) : mfma16(g2, q[v][p], acc);
      acc = tall ? mfma16(q[v][p], g, acc) : mfma16(g, q[v][p], acc);
    }
    return acc;
  };
  if (J.y_tall) {
    for (int j = 16 * cg; j < nc; j += 16 * CG) {
      f32x4_t acc = {0, 0, 0, 0};
#pragma unroll
      for (int v = 0; v < NT / K2; ++v) acc = dot(v, j + lo, true, acc);
      acc = acc * scale;
      const int i = 16 * t + 4 * hi;   // rows i + m, column j + lo
      if (j + lo < nc) st_run16<DT, 4>(y + (int64_t)(j0 + j + lo) * J.r + i, J.r - i, (const float*)&acc);
    }
  } else {
    for (int j = 32 * cg; j < nc; j += 32 * CG) {
      f32x4_t acc[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
      const int c = j + 8 * (lo >> 2) + (lo & 3);   // row 4 hi + m of the pair's results: columns 8 hi + m and 8 hi + 4 + m
#pragma unroll
      for (int v = 0; v < NT / K2; ++v) {
        acc[0] = dot(v, c, false, acc[0]);
        acc[1] = dot(v, c + 4, false, acc[1]);
      }
      acc[0] = acc[0] * scale;
      acc[1] = acc[1] * scale;
      const int i = 16 * t + lo, k = j + 8 * hi;   // row i, columns k to k + 7
      if (i < J.r) st_run16<DT, 8>(y + (int64_t)i * J.n + j0 + k, nc - k, (const float*)acc);
    }
  }
}

// ------------------------------------------------------------------------------------------------ steps of r > 64, as launches

constexpr int BIG = 8, BIG_MAT = BIG * BIG * 256;   // doubles of a matrix: 64 tiles in the operand layout
struct BigArgs {
  const double* part;
  double *A, *P, *T, *Q, *Q2;   // [mats][BIG_MAT]
  double *tr, *qscale;          // [mats][8], [mats]
  int mats;
  int first, last;
  Steps st;
};
// blocks of a matrix to one XCD, whose L2 then holds its tiles: block b -> matrix, index among the matrix's `n` blocks
SMEL_DEV bool big_map(int mats, int n, int& mat, int& k) {
  const int x = blockIdx.x % NXCD, j = blockIdx.x / NXCD;
  mat = j / n * NXCD + x;
  k = j % n;
  return mat < mats;
}

// tile (t, u) of M N for symmetric M and N that commute
SMEL_DEV f64x4_t big_product(const double* M, const double* N, int t, int u, int lane) {
  f64x4_t a[BIG], b[BIG], acc = {0, 0, 0, 0};
#pragma unroll
  for (int k = 0; k < BIG; ++k) {
    a[k] = *(const f64x4_t*)(M + ((k * BIG + t) * 64 + lane) * 4);
    b[k] = *(const f64x4_t*)(N + ((k * BIG + u) * 64 + lane) * 4);
  }
  __builtin_amdgcn_sched_barrier(0);   // every load is on its way before the first product
#pragma unroll
  for (int k = 0; k < BIG; ++k)
#pragma unroll
    for (int m = 0; m < 4; ++m) acc = mfma64(a[k][m], b[k][m], acc);
  return acc;
}

// tile (t, u), t <= u, and its mirror (through the wave's own LDS tile, in the wave's order)
SMEL_DEV void big_store(double* M, int t, int u, int lane, f64x4_t v, double* l) {
  const int lo = lane & 15, hi = lane >> 4;
  *(f64x4_t*)(M + ((t * BIG + u) * 64 + lane) * 4) = v;
  if (t == u) return;
#pragma unroll
  for (int m = 0; m < 4; ++m) l[(4 * m + hi) * TP + lo] = v[m];
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  f64x4_t b;
#pragma unroll
  for (int m = 0; m < 4; ++m) b[m] = l[lo * TP + 4 * m + hi];
  *(f64x4_t*)(M + ((u * BIG + t) * 64 + lane) * 4) = b;
}

// the parts' sum as A0, and the diagonal tiles' traces; here and below a wave per upper tile
__global__ __launch_bounds__(256) void big_sum_kernel(Jobs js, BigArgs g) {
  constexpr int NTL = ntiles(BIG);
  __shared__ double tile[4][16 * TP];
  int mat, kb;
  if (!big_map(g.mats, NTL / 4, mat, kb)) return;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, lo = lane & 15, hi = lane >> 4;
  const Job& J = js.j[find_job<BY_MATRIX>(js, mat)];
  int t, u;
  tile_of(kb * 4 + wave, BIG, t, u);
  const double* const p = g.part + (J.part0 + (int64_t)(mat - J.mat0) * J.parts) * (NTL * 256) + ((kb * 4 + wave) * 64 + lane) * 4;
  f64x4_t a = {0, 0, 0, 0};
#pragma unroll 8
  for (int s = 0; s < J.parts; ++s) a += *(const f64x4_t*)(p + (int64_t)s * (NTL * 256));
  big_store(g.A + (int64_t)mat * BIG_MAT, t, u, lane, a, tile[wave]);
  if (t == u) {
    double d = 0;
#pragma unroll
    for (int m = 0; m < 4; ++m) d += 4 * m + hi == lo ? a[m] : 0.0;
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) d += __shfl_xor(d, o, 64);
    if (lane == 0) g.tr[mat * BIG + t] = d;
  }
}

// BIG_P: P = a I + b A + c A A (first: of the scaled A, and Q = s P);  BIG_TQ: T = A P and Q2 = P Q;  BIG_A: A = T P
enum { BIG_P, BIG_TQ, BIG_A };
template <int WHAT>
__global__ __launch_bounds__(256, 2) void big_kernel(BigArgs g) {
  constexpr int NTL = ntiles(BIG);
  __shared__ double tile[4][16 * TP];
  int mat, kb;
  if (!big_map(g.mats, NTL / 4, mat, kb)) return;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, lo = lane & 15, hi = lane >> 4;
  int t, u;
  tile_of(kb * 4 + wave, BIG, t, u);
  const int64_t base = (int64_t)mat * BIG_MAT, at = base + ((t * BIG + u) * 64 + lane) * 4;
  double s = 1.0;
  if (g.first) {   // the trace is the squared norm
    double tr = 0;
#pragma unroll
    for (int i = 0; i < BIG; ++i) tr += g.tr[mat * BIG + i];
    s = inv_norm(g.st, tr);
  }
  const double s2 = s * s;
  if constexpr (WHAT == BIG_P) {
    f64x4_t p;
#pragma unroll
    for (int m = 0; m < 4; ++m) p[m] = t == u && 4 * m + hi == lo ? 1.0 : 0.0;
    if (g.st.steps > 0) {
      const f64x4_t aa = big_product(g.A + base, g.A + base, t, u, lane);
      p = g.st.a * p + g.st.b * (*(const f64x4_t*)(g.A + at) * s2) + g.st.c * (aa * s2 * s2);
      big_store(g.P + base, t, u, lane, p, tile[wave]);
    }
    if (g.first) {
      const int ex = exp_of(s);
      big_store(g.Q + base, t, u, lane, p * ldexp(s, -ex), tile[wave]);
      if (kb == 0 && threadIdx.x == 0) g.qscale[mat] = ldexp(1.0, ex);
    }
  } else if constexpr (WHAT == BIG_TQ) {
    if (blockIdx.y == 0 && !g.last) big_store(g.T + base, t, u, lane, big_product(g.A + base, g.P + base, t, u, lane) * s2, tile[wave]);
    if (!g.first && (blockIdx.y == 1 || g.last))
      big_store(g.Q2 + base, t, u, lane, big_product(g.P + base, g.Q + base, t, u, lane), tile[wave]);
  } else {
    big_store(g.A + base, t, u, lane, big_product(g.T + base, g.P + base, t, u, lane), tile[wave]);
  }
}

// ------------------------------------------------------------------------------------------------ passes on X in 64 bits

// X: a group's matrices one after the other, each as blocks [n / 16][16 NT rows][16 columns], zero past r and n: what the matrix
// instruction takes of a block lies together.
SMEL_DEV double* x64_of(const Jobs& js, int k, int mat, int nt, double* X) {
  int64_t at = 0;
  for (int q = 0; q < k; ++q) at += (int64_t)js.j[q].batch * ((js.j[q].n + 15) >> 4);
  return X + (at + (int64_t)mat * ((js.j[k].n + 15) >> 4)) * (256 * nt);
}

// The parts of X X^T, as gram_kernel's: a block's columns, tiles dealt to the waves (at r = 128 as there). A tile's operand is 2 KB in
// one piece, which the rows' other tiles find in the caches. Every element is one chain of products in column order, so equal rows
// give equal elements. 36 x 128 x 2816: 51 us (27 of f64 products).
constexpr int gram64_waves(int nt) { return nt == 8 ? 12 : nt == 4 ? 5 : ntiles(nt); }
template <int NT>
__global__ __launch_bounds__(64 * gram64_waves(NT)) void gram64_kernel(Jobs js, const double* __restrict__ X, double* __restrict__ part) {
  constexpr int NTL = ntiles(NT), W = gram64_waves(NT), TPW = NTL / W;
  static_assert(TPW * W == NTL, "tiles per wave");
  const int k = find_job<BY_GRAM>(js, blockIdx.x);
  const Job& J = js.j[k];
  const int lb = blockIdx.x - J.gblk0, mat = lb / J.parts;
  const int b0 = lb % J.parts * (js.per >> 4), b1 = min(b0 + (js.per >> 4), (J.n + 15) >> 4);
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, lo = lane & 15, hi = lane >> 4;
  const double* const x = x64_of(js, k, mat, NT, const_cast<double*>(X)) + lo * 16 + hi * 4;
  auto operand = [&](int64_t b, int tile) { return *(const f64x4_t*)(x + (b * NT + tile) * 256); };
  f64x4_t acc[TPW];
  int tile[TPW];
#pragma unroll
  for (int q = 0; q < TPW; ++q) acc[q] = f64x4_t{0, 0, 0, 0};
  if constexpr (NT == 8) {
    const uint32_t rows = GRAM_ROWS[wave];
    const int ra = rows >> 8, rb = rows >> 4 & 15, rc = rows & 15;
    if (wave < 8) {
      tile[0] = tile_at(ra, rb, NT);
      tile[1] = tile_at(ra, rc, NT);
      tile[2] = tile_at(rb, rc, NT);
      f64x4_t an = operand(b0, ra), bn = operand(b0, rb), cn = operand(b0, rc);
      for (int j = b0; j < b1; ++j) {   // the next block's on their way
        const f64x4_t a = an, b = bn, c = cn;
        const int next = min(j + 1, b1 - 1);
        an = operand(next, ra), bn = operand(next, rb), cn = operand(next, rc);
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          acc[0] = mfma64(a[m], b[m], acc[0]);
          acc[1] = mfma64(a[m], c[m], acc[1]);
          acc[2] = mfma64(b[m], c[m], acc[2]);
        }
      }
    } else {
      tile[0] = tile_at(ra, rb, NT);
      tile[1] = tile_at(ra, ra, NT);
      tile[2] = tile_at(rb, rb, NT);
      f64x4_t an = operand(b0, ra), bn = operand(b0, rb);
      for (int j = b0; j < b1; ++j) {
        const f64x4_t a = an, b = bn;
        const int next = min(j + 1, b1 - 1);
        an = operand(next, ra), bn = operand(next, rb);
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          acc[0] = mfma64(a[m], b[m], acc[0]);
          acc[1] = mfma64(a[m], a[m], acc[1]);
          acc[2] = mfma64(b[m], b[m], acc[2]);
        }
      }
    }
  } else {
    int t[TPW], u[TPW];
#pragma unroll
    for (int q = 0; q < TPW; ++q) {
      tile[q] = wave * TPW + q;
      tile_of(tile[q], NT, t[q], u[q]);
    }
    f64x4_t an[TPW], bn[TPW];
#pragma unroll
    for (int q = 0; q < TPW; ++q) an[q] = operand(b0, t[q]), bn[q] = operand(b0, u[q]);
    for (int j = b0; j < b1; ++j) {
      const int next = min(j + 1, b1 - 1);
#pragma unroll
      for (int q = 0; q < TPW; ++q) {
        const f64x4_t a = an[q], b = bn[q];
        an[q] = operand(next, t[q]), bn[q] = operand(next, u[q]);
#pragma unroll
        for (int m = 0; m < 4; ++m) acc[q] = mfma64(a[m], b[m], acc[q]);
      }
    }
  }
#pragma unroll
  for (int q = 0; q < TPW; ++q) *(f64x4_t*)(part + ((J.part0 + lb) * (int64_t)NTL + tile[q]) * 256 + lane * 4) = acc[q];
}

// the steps of r <= 32, a block per matrix: Q's tiles to memory
template <int NT>
__global__ __launch_bounds__(64 * WAVES) void steps_kernel(Jobs js, Steps st, const double* __restrict__ part,
                                                           double* __restrict__ Qout, double* __restrict__ qscale) {
  constexpr int N2 = NT * NT;
  __shared__ f64x4_t b[4 * N2][64];
  __shared__ double tr[NT];
  const Job& J = js.j[find_job<BY_MATRIX>(js, blockIdx.x)];
  const double scale = steps_small<NT>(J, blockIdx.x - J.mat0, st, part, b, tr);
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  if (wave < N2) *(f64x4_t*)(Qout + ((int64_t)blockIdx.x * N2 + wave) * 256 + lane * 4) = b[3 * N2 + wave][lane];
  if (threadIdx.x == 0) qscale[blockIdx.x] = scale;
}

enum { X64 = 3 };   // beside the types 0 to 2: the group's X
SMEL_DEV double ld_as(const void* p, int64_t i, int dt) {
  switch (dt) {
    case 0: return __uint_as_float((uint32_t)((const uint16_t*)p)[i] << 16);
    case 1: return ((const float*)p)[i];
    case 2: return (float)((const _Float16*)p)[i];
    default: return ((const double*)p)[i];
  }
}
// A 16-bit value is rounded by way of fp32: off by 2^-16 (bf16), 2^-13 (fp16) of its half step more at most
SMEL_DEV void st_as(void* p, int64_t i, int dt, double v) {
  switch (dt) {
    case 0: ((uint16_t*)p)[i] = f2bf((float)v); break;
    case 1: ((float*)p)[i] = (float)v; break;
    case 2: ((_Float16*)p)[i] = (_Float16)(float)v; break;
    default: ((double*)p)[i] = v;
  }
}

// alpha X + Q X from `in` (G's type, or X64) to `out` (the result's type, or X64: in place). A wave owns a tile of rows, whose part of
// Q stays in registers, and every CG-th block of 16 columns; the block's columns pass through LDS, the next ones on their way while
// some are multiplied. A register of a lane is the operand's and the result's element alike. 36 x 128 x 2816: 92 us, 41 of bytes;
// a step of the formula 160 (390 with X in rows of n and Q read for every 16 columns by every wave).
template <int NT>
__global__ __launch_bounds__(64 * WAVES) void apply64_kernel(Jobs js, double alpha, const double* __restrict__ Q,
                                                             const double* __restrict__ qscale, double* X, int in, int out) {
  constexpr int CG = WAVES / NT, RP = 16 * NT, PER = 4;   // elements of a thread: CG RP 16 / (64 WAVES)
  __shared__ double buf[2][CG * RP * 16];
  const int k = find_job<BY_APPLY>(js, blockIdx.x);
  const Job& J = js.j[k];
  const int lb = blockIdx.x - J.blk0, mat = lb / J.slices, j0 = (lb % J.slices) << js.lg;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, lo = lane & 15, hi = lane >> 4, t = wave % NT, cg = wave / NT;
  const int nc = min(1 << js.lg, J.n - j0);
  double* const x64 = x64_of(js, k, mat, NT, X) + (int64_t)(j0 >> 4) * (RP * 16);
  double v[PER];
  // element e of CG column blocks from column c on: its place in LDS
  auto place = [&](int q) {
    const int e = threadIdx.x + q * 64 * WAVES;
    return in != X64 && J.x_tall ? e / (RP * 16) * (RP * 16) + e % RP * 16 + e / RP % 16 : e;
  };
  auto fetch = [&](int c) {
#pragma unroll
    for (int q = 0; q < PER; ++q) {
      const int at = place(q), i = at / 16 % RP, col = c + at / (RP * 16) * 16 + at % 16;
      v[q] = 0;
      if (in == X64) {
        if (col < ((nc + 15) & ~15)) v[q] = x64[(int64_t)c * RP + at];
      } else if (i < J.r && col < nc) {
        const int64_t j = j0 + col;
        v[q] = ld_as(J.x, mat * J.xb + (J.x_tall ? j * J.ld + i : i * J.ld + j), in);
      }
    }
  };
  fetch(0);
  f64x4_t q[NT];
  const double scale = qscale[J.mat0 + mat];
#pragma unroll
  for (int u = 0; u < NT; ++u) q[u] = *(const f64x4_t*)(Q + (int64_t)(J.mat0 + mat) * (NT * NT * 256) + ((u * NT + t) * 64 + lane) * 4) * scale;
  for (int c = 0, par = 0; c < nc; c += 16 * CG, par ^= 1) {
    double* const b = buf[par];
#pragma unroll
    for (int e = 0; e < PER; ++e) b[place(e)] = v[e];
    __syncthreads();   // the buffers alternate: who reads b has passed the next barrier before it is written again
    if (c + 16 * CG < nc) fetch(c + 16 * CG);
    const int w = c + 16 * cg;
    if (w >= nc) continue;
    const double* const x = b + cg * (RP * 16);
    f64x4_t acc = {0, 0, 0, 0}, own;
#pragma unroll
    for (int u = 0; u < NT; ++u)
#pragma unroll
      for (int m = 0; m < 4; ++m) acc = mfma64(q[u][m], x[(16 * u + 4 * m + hi) * 16 + lo], acc);
#pragma unroll
    for (int m = 0; m < 4; ++m) own[m] = fma(alpha, x[(16 * t + 4 * m + hi) * 16 + lo], acc[m]);
    if (out == X64) {
#pragma unroll
      for (int m = 0; m < 4; ++m) x64[(int64_t)w * RP + (16 * t + 4 * m + hi) * 16 + lo] = own[m];
    } else {
      const int64_t j = j0 + w + lo;
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        const int64_t i = 16 * t + 4 * m + hi;
        if (w + lo < nc && i < J.r) st_as(J.y, (int64_t)mat * J.r * J.n + (J.y_tall ? j * J.r + i : i * J.n + j), out, own[m]);
      }
    }
  }
}

// ------------------------------------------------------------------------------------------------ host

int nt_of(int64_t r) { return r <= 16 ? 1 : r <= 32 ? 2 : r <= 64 ? 4 : 8; }

int check(const smel_ortho_job* jobs, int32_t n) {
  SMEL_REQUIRE(n >= 0 && (jobs || n == 0), SMEL_EINVAL, "orthogonalize: null jobs");
  for (int k = 0; k < n; ++k) {
    const smel_ortho_job& j = jobs[k];
    SMEL_REQUIRE(j.batch >= 0 && j.rows >= 0 && j.cols >= 0, SMEL_EINVAL, "orthogonalize: job %d has a negative size", k);
    if (j.batch == 0 || j.rows == 0 || j.cols == 0) continue;
    SMEL_REQUIRE(j.rows <= MAX_R || j.cols <= MAX_R, SMEL_EUNSUPPORTED,
                 "orthogonalize: a %lld x %lld matrix, the short side is at most %d", (long long)j.rows, (long long)j.cols, MAX_R);
    SMEL_REQUIRE(j.rows < (int64_t)1 << 30 && j.cols < (int64_t)1 << 30 && j.batch < (int64_t)1 << 30, SMEL_EUNSUPPORTED,
                 "orthogonalize: job %d has a side of 2^30 or more", k);
    SMEL_REQUIRE(j.dtype >= 0 && j.dtype <= 2, SMEL_EINVAL, "orthogonalize: dtype %lld (0 = bf16, 1 = fp32, 2 = fp16)",
                 (long long)j.dtype);
    SMEL_REQUIRE(j.x && j.y, SMEL_EINVAL, "orthogonalize: null pointer");
    const int es = j.dtype == 1 ? 4 : 2;
    SMEL_REQUIRE((uintptr_t)j.x % es == 0 && (uintptr_t)j.y % es == 0, SMEL_EINVAL, "orthogonalize: misaligned pointer");
    SMEL_REQUIRE(j.x_row >= 0 && j.x_col >= 0 && j.x_batch >= 0, SMEL_EINVAL, "orthogonalize: negative stride");
    SMEL_REQUIRE((j.cols == 1 || j.x_col == 1) || (j.rows == 1 || j.x_row == 1), SMEL_EINVAL,
                 "orthogonalize: neither side of job %d has unit stride", k);
  }
  return 0;
}

struct Plan {
  Jobs js;
  int64_t blocks, gblocks, mats;   // apply's and gram's blocks, matrices
};
struct Cursor {
  int job;
  int64_t mat;
};
constexpr int64_t MAX_MATS = 65536, BIG_MATS = 256;   // of a launch; its workspace is 0.6 MB a matrix above r = 64
constexpr int64_t MAX_PIECES = 1 << 21;               // of 128 columns: a launch takes fewer than 2^32 threads

// the next jobs of one (tiles a side, dtype) from `at` on, as many as a launch takes (a job's batch may be split)
Cursor fill(const smel_ortho_job* jobs, int32_t n, Cursor at, int nt, int dt, Plan& p) {
  p.js.n = 0;
  p.blocks = p.gblocks = p.mats = 0;
  struct Taken {
    int job;
    int64_t mat, count;
  } taken[MAX_JOBS];
  int64_t cols = 0, pieces = 0;
  const int64_t most = nt == 8 ? BIG_MATS : MAX_MATS;
  while (at.job < n && p.js.n < MAX_JOBS && p.mats < most) {
    const smel_ortho_job& j = jobs[at.job];
    const int64_t r = j.rows < j.cols ? j.rows : j.cols;
    if (j.batch == 0 || r == 0 || j.dtype != dt || nt_of(r) != nt) {
      at = Cursor{at.job + 1, 0};
      continue;
    }
    const int64_t of_one = ((j.rows < j.cols ? j.cols : j.rows) + 127) / 128;
    if (pieces && pieces + of_one > MAX_PIECES) break;
    const int64_t take = std::min({j.batch - at.mat, most - p.mats, std::max<int64_t>((MAX_PIECES - pieces) / of_one, 1)});
    pieces += take * of_one;
    taken[p.js.n++] = Taken{at.job, at.mat, take};
    p.mats += take;
    cols += take * (j.rows < j.cols ? j.cols : j.rows);
    at.mat += take;
    if (at.mat == j.batch) at = Cursor{at.job + 1, 0};
  }
  // the largest slices that give most CUs a block, but at least 128 columns (each wave a block of 16); up to r = 32 every
  // block runs the steps, and two on a CU get in each other's way (a layer's 84 updates: 20.7 us with 780 blocks, 14.4 with 195)
  int slice = dt == 1 ? max_slice(nt) : max_slice16(nt);
  while (slice > 128 && cols / slice < 192) slice /= 2;
  p.js.lg = __builtin_ctz(slice);
  // gram: likewise, down to 64 columns at r > 64; then one round of blocks (two on a CU, one at r > 64, whose blocks fill it
  // and whose parts are 72 KB each)
  int gs = gram_slice(nt);
  while (gs > 128 && cols / gs < 512) gs /= 2;
  p.js.glg = __builtin_ctz(gs);
  const int64_t round = nt == 8 ? 256 : 512;
  p.js.per = (int)std::max<int64_t>(gs, std::min<int64_t>(cols / round / 16 * 16, 1 << 30));
  for (;;) {
    int64_t blocks = 0;
    for (int k = 0; k < p.js.n; ++k) {
      const smel_ortho_job& j = jobs[taken[k].job];
      const int64_t n = j.rows < j.cols ? j.cols : j.rows;
      blocks += taken[k].count * ((n + p.js.per - 1) / p.js.per);
    }
    if (blocks <= round || blocks <= p.mats) break;   // or a block a matrix
    p.js.per += std::max(16, p.js.per / 256 * 16);
  }
  int64_t mats = 0;
  for (int k = 0; k < p.js.n; ++k) {
    const smel_ortho_job& j = jobs[taken[k].job];
    Job& o = p.js.j[k];
    const bool wide = j.rows <= j.cols;   // the short side is the rows
    const int64_t es = dt == 1 ? 4 : 2;
    o.x = (const char*)j.x + taken[k].mat * j.x_batch * es;
    o.y = (char*)j.y + taken[k].mat * j.rows * j.cols * es;
    o.xb = j.x_batch;
    o.r = (int32_t)(wide ? j.rows : j.cols);
    o.n = (int32_t)(wide ? j.cols : j.rows);
    o.batch = (int32_t)taken[k].count;
    o.y_tall = !wide;
    const bool last = j.cols == 1 || j.x_col == 1;   // lines run along the last side
    if (last && !(j.cols == 1 && j.rows > 1 && j.x_row == 1)) {
      o.ld = j.x_row;
      o.x_tall = !wide;
    } else {
      o.ld = j.x_col;
      o.x_tall = wide;
    }
    o.slices = (o.n + slice - 1) / slice;
    o.parts = (o.n + p.js.per - 1) / p.js.per;
    o.blk0 = (int32_t)p.blocks;
    o.gblk0 = (int32_t)p.gblocks;
    o.mat0 = (int32_t)mats;
    o.part0 = p.gblocks;
    mats += o.batch;
    p.blocks += (int64_t)o.batch * o.slices;
    p.gblocks += (int64_t)o.batch * o.parts;
    if (p.blocks >= (int64_t)1 << 22) return Cursor{-1, 0};   // one matrix of 2^29 columns or more, r > 32
  }
  return at;
}

// steps of a pass on the r x r matrices: their rounding grows by a^2 a step
int pass_steps(double a) {
  const double growth = std::max(1.0, a * a);
  int k = 1;
  for (double g = growth * growth; k < 64 && g <= 0x1p24; g *= growth) ++k;
  return k;
}

int64_t part_bytes(const Plan& p, int nt) { return p.gblocks * ntiles(nt) * 2048; }
// of the r x r matrices beside Q's tiles and scale: none to r = 64
int64_t q_bytes(const Plan& p, int nt) {
  return nt == 8 ? p.mats * (5 * BIG_MAT + BIG + 1) * 8 : p.mats * (nt * nt * 256 + 1) * 8;
}
int64_t ws_bytes_of(const Plan& p, int nt, bool passes) {
  const int64_t parts = part_bytes(p, nt);
  if (!passes) return nt <= 2 ? parts : parts + q_bytes(p, nt);
  int64_t blocks = 0;   // of X
  for (int k = 0; k < p.js.n; ++k) blocks += (int64_t)p.js.j[k].batch * ((p.js.j[k].n + 15) >> 4);
  return parts + (q_bytes(p, nt) + 31) / 32 * 32 + blocks * (256 * nt * 8);
}

// the steps above r = 64; returns where Q's tiles are
const double* run_big(const Plan& p, const Steps& st, const double* part, double* ws, const double*& qscale,
                      hipStream_t stream) {
  BigArgs g{};
  const int64_t m = p.mats * BIG_MAT;
  g.part = part;
  g.A = ws;
  g.P = ws + m;
  g.T = ws + 2 * m;
  g.Q = ws + 3 * m;
  g.Q2 = ws + 4 * m;
  g.tr = ws + 5 * m;
  qscale = g.qscale = g.tr + p.mats * BIG;
  g.mats = (int)p.mats;
  g.st = st;
  const unsigned groups = (unsigned)((p.mats + NXCD - 1) / NXCD * NXCD);
  big_sum_kernel<<<groups * (ntiles(BIG) / 4), 256, 0, stream>>>(p.js, g);
  for (int it = 0; it == 0 || it < st.steps; ++it) {
    g.first = it == 0;
    g.last = it + 1 >= st.steps;
    big_kernel<BIG_P><<<groups * (ntiles(BIG) / 4), 256, 0, stream>>>(g);
    if (g.first && g.last) break;
    big_kernel<BIG_TQ><<<dim3(groups * (ntiles(BIG) / 4), g.first || g.last ? 1 : 2), 256, 0, stream>>>(g);
    if (!g.first) std::swap(g.Q, g.Q2);
    if (!g.last) big_kernel<BIG_A><<<groups * (ntiles(BIG) / 4), 256, 0, stream>>>(g);
  }
  return g.Q;
}

// Q's tiles from the parts: where they are, and their scale
template <int NT>
const double* run_steps(const Plan& p, const Steps& st, const double* part, double* rest, const double*& qscale,
                        hipStream_t stream) {
  if constexpr (NT == 8) {
    return run_big(p, st, part, rest, qscale, stream);
  } else {
    double* const scale = rest + p.mats * NT * NT * 256;
    if constexpr (NT == 4) iterate_kernel<<<(unsigned)p.mats, 64 * IT_WAVES, 0, stream>>>(p.js, st, part, rest, scale);
    else steps_kernel<NT><<<(unsigned)p.mats, 64 * WAVES, 0, stream>>>(p.js, st, part, rest, scale);
    qscale = scale;
    return rest;
  }
}

template <int NT, int DT, bool SMALL>
void run_apply(const Plan& p, const Steps& st, const double* in, const double* qscale, hipStream_t stream) {
  if constexpr (DT == 1) apply_kernel<NT, SMALL><<<(unsigned)p.blocks, 64 * WAVES, 0, stream>>>(p.js, st, in, qscale);
  else apply16_kernel<NT, DT, SMALL><<<(unsigned)p.blocks, 64 * WAVES, 0, stream>>>(p.js, st, in, qscale);
}
template <int NT, int DT>
int run(const Plan& p, const Steps& st, void* ws, hipStream_t stream) {
  const Jobs& js = p.js;
  double* const part = (double*)ws;
  double* const rest = (double*)((char*)ws + part_bytes(p, NT));
  gram_kernel<NT, DT><<<(unsigned)p.gblocks, 64 * gram_waves(NT), 0, stream>>>(js, part);
  if constexpr (NT <= 2) {
    run_apply<NT, DT, true>(p, st, part, nullptr, stream);
  } else {
    const double* qscale = nullptr;
    const double* const Q = run_steps<NT>(p, st, part, rest, qscale, stream);
    run_apply<NT, DT, false>(p, st, Q, qscale, stream);
  }
  return smel::launch_status();
}
// More steps than a pass takes
template <int NT, int DT>
int run_passes(const Plan& p, const Steps& st, int most, void* ws, hipStream_t stream) {
  double* const part = (double*)ws;
  double* const rest = (double*)((char*)ws + part_bytes(p, NT));
  double* const X = (double*)((char*)rest + (q_bytes(p, NT) + 31) / 32 * 32);
  auto pass = [&](bool first, bool last, const Steps& s, double alpha) {
    if (first) gram_kernel<NT, DT><<<(unsigned)p.gblocks, 64 * gram_waves(NT), 0, stream>>>(p.js, part);
    else gram64_kernel<NT><<<(unsigned)p.gblocks, 64 * gram64_waves(NT), 0, stream>>>(p.js, X, part);
    const double* qscale = nullptr;
    const double* const Q = run_steps<NT>(p, s, part, rest, qscale, stream);
    apply64_kernel<NT><<<(unsigned)p.blocks, 64 * WAVES, 0, stream>>>(p.js, alpha, Q, qscale, X, first ? DT : X64, last ? DT : X64);
  };
  if (st.steps <= 2 * most) {
    pass(true, false, Steps{(st.steps + 1) / 2, 0, st.a, st.b, st.c, st.eps}, 0);
    pass(false, true, Steps{st.steps / 2, 1, st.a, st.b, st.c, 0}, 0);
  } else {   // X0, then a step each: Q = b A + c A^2
    pass(true, false, Steps{0, 0, st.a, st.b, st.c, st.eps}, 0);
    for (int it = 0; it < st.steps; ++it) pass(false, it + 1 == st.steps, Steps{1, 1, 0, st.b, st.c, 0}, st.a);
  }
  return smel::launch_status();
}
template <int NT>
int run_dt(const Plan& p, int dt, const Steps& st, void* ws, hipStream_t stream) {
  if (const int most = pass_steps(st.a); st.steps > most)
    return dt == 0 ? run_passes<NT, 0>(p, st, most, ws, stream) : dt == 1 ? run_passes<NT, 1>(p, st, most, ws, stream)
                                                                          : run_passes<NT, 2>(p, st, most, ws, stream);
  return dt == 0 ? run<NT, 0>(p, st, ws, stream) : dt == 1 ? run<NT, 1>(p, st, ws, stream) : run<NT, 2>(p, st, ws, stream);
}

// f(plan, nt, dt) for every launch group, in order; stops at the first non-zero result
template <class F>
int each(const smel_ortho_job* jobs, int32_t n, F f) {
  bool any[9][3] = {};
  for (int k = 0; k < n; ++k) {
    const int64_t r = jobs[k].rows < jobs[k].cols ? jobs[k].rows : jobs[k].cols;
    if (jobs[k].batch && r) any[nt_of(r)][jobs[k].dtype] = true;
  }
  for (int nt = 1; nt <= 8; nt *= 2)
    for (int dt = 0; dt < 3; ++dt)
      for (Cursor at{0, 0}; any[nt][dt] && at.job < n;) {
        Plan p;
        at = fill(jobs, n, at, nt, dt, p);
        SMEL_REQUIRE(at.job >= 0, SMEL_EUNSUPPORTED, "orthogonalize: a matrix has too many columns for one launch");
        if (p.js.n == 0) continue;
        const int rc = f(p, nt, dt);
        if (rc) return rc;
      }
  return 0;
}

int64_t ws_need(const smel_ortho_job* jobs, int32_t n, bool passes, int& rc) {
  int64_t need = 0;   // the groups run one after the other on one stream and share the workspace
  rc = each(jobs, n, [&](const Plan& p, int nt, int) {
    need = std::max(need, ws_bytes_of(p, nt, passes));
    return 0;
  });
  return need;
}

}  // namespace

extern "C" int64_t smel_orthogonalize_ws(const smel_ortho_job* jobs, int32_t n_jobs, int32_t steps, double a) {
  if (check(jobs, n_jobs)) return -1;
  int rc = 0;
  const int64_t need = ws_need(jobs, n_jobs, steps > pass_steps(a), rc);
  return rc ? -1 : need;
}

extern "C" int smel_orthogonalize(const smel_ortho_job* jobs, int32_t n_jobs, int32_t steps, double a, double b,
                                  double c, double eps, void* ws, int64_t ws_bytes, hipStream_t stream) {
  int rc = check(jobs, n_jobs);
  if (rc) return rc;
  SMEL_REQUIRE(steps >= 0 && steps <= 64, SMEL_EINVAL, "orthogonalize: %d steps (0 to 64)", steps);
  SMEL_REQUIRE(eps >= 0, SMEL_EINVAL, "orthogonalize: eps %g", eps);
  const int64_t need = ws_need(jobs, n_jobs, steps > pass_steps(a), rc);
  if (rc) return rc;
  SMEL_REQUIRE(need == 0 || (ws && (uintptr_t)ws % 16 == 0 && ws_bytes >= need), SMEL_EINVAL,
               "orthogonalize: a workspace of %lld bytes, 16-byte aligned, is needed (got %lld)", (long long)need,
               (long long)ws_bytes);
  const Steps st{steps, 0, a, b, c, eps};
  return each(jobs, n_jobs, [&](const Plan& p, int nt, int dt) {
    return nt == 1 ? run_dt<1>(p, dt, st, ws, stream) : nt == 2 ? run_dt<2>(p, dt, st, ws, stream)
           : nt == 4 ? run_dt<4>(p, dt, st, ws, stream) : run_dt<8>(p, dt, st, ws, stream);
  });
}
